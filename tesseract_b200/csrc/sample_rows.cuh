// How tb_sample cuts a row among blocks: sampling.cu launches by it, and token_choice.cu finds with it the token that sampling.cu gives a
// row with logits that are not finite.
#pragma once

#include "common.cuh"

constexpr int kSampleThreads = 1024;

// Blocks per row: as many (a power of two up to the portable cluster size) as keep the grid within one wave.
static inline int sample_blocks(int rows, int vocab) {
    static int sms = 0;
    if (sms == 0) {
        int device = 0;
        cudaGetDevice(&device);
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 1;
    }
    int blocks = 8;
    while (blocks > 1 && (rows * blocks > sms || vocab < blocks * kSampleThreads)) blocks >>= 1;
    return blocks;
}

// Tokens of a block.
static inline int sample_chunk(int blocks, int vocab) {
    return ((vocab + blocks - 1) / blocks + kSampleThreads - 1) / kSampleThreads * kSampleThreads;
}
