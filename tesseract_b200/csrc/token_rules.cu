// Histories of tokens a request, and logits under a request's rules (token_rules.cuh).
#include "token_rules.cuh"

namespace {

// ---- histories
//
// seen: a bit for every token of the prompt and the answer; counts: how often the answer has each.  A history begun anew (the requests
// whose first tokens a step brings) writes 4 V + V / 8 bytes: 32 requests of 512 tokens over 128,256 take 6.4 us on the device, of up to
// 8,192 tokens 8.3, of which 4.8 remain when no block goes through the tokens (17 MB are 2.7 us at the copy rate); one request 2.8 us, a
// launch and three dependent loads.  Tokens added to histories that are there (later portions, decode steps) touch two sectors each: 32
// portions of 512 tokens 2.0 us, a token a row 1.4 for 1 to 32 rows, a launch and what the loads and atomics take to come back.

constexpr int kNoteThreads = 512;
constexpr int kNotePart = 8192;          // tokens of the vocabulary that a block begins anew

// grid (parts of the vocabulary, rows): a slot's history in place of what stands there.  Every block goes through all of its row's tokens
// (from L2, but for the first) and counts those of its part in shared memory, so that a part is written once, whole.  Of rows that name
// one slot the last counts.
__global__ void __launch_bounds__(kNoteThreads)
restart_kernel(uint32_t* __restrict__ seen, int* __restrict__ counts, int slot_count, int words, int stride, int vocab,
               const int* __restrict__ slots, const int* __restrict__ tokens, int total, const int* __restrict__ starts,
               const int* __restrict__ prompts, int rows) {
    __shared__ __align__(16) int times[kNotePart];
    __shared__ __align__(16) uint32_t bits[kNotePart / 32];
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.y, t = threadIdx.x, slot = slots[row];
    if (slot < 0 || slot >= slot_count) return;
    int later = 0;
    for (int r = row + 1 + t; r < rows; r += kNoteThreads) later |= slots[r] == slot;
    for (int i = t; i < kNotePart / 4; i += kNoteThreads) reinterpret_cast<int4*>(times)[i] = make_int4(0, 0, 0, 0);
    if (t < kNotePart / 32) bits[t] = 0;
    if (__syncthreads_or(later)) return;
    const int first = blockIdx.x * kNotePart;
    const int begin = starts != nullptr ? max(0, starts[row]) : row;
    const int end = starts != nullptr ? min(total, starts[row + 1]) : row + 1;
    const int prompt = prompts != nullptr ? prompts[row] : 0;
#pragma unroll 4
    for (int i = begin + t; i < end; i += kNoteThreads) {
        const unsigned at = (unsigned)tokens[i] - (unsigned)first;     // (a token below the part, or negative, is beyond it as well)
        if (at >= (unsigned)kNotePart || (int)at + first >= vocab) continue;
        atomicOr(bits + (at >> 5), 1u << (at & 31));
        if (i - begin >= prompt) atomicAdd(times + at, 1);
    }
    __syncthreads();
    // (rows of both are multiples of 16 bytes)
    int4* to = reinterpret_cast<int4*>(counts + (int64_t)slot * stride + first);
    for (int i = t; i < min(kNotePart, stride - first) / 4; i += kNoteThreads) to[i] = reinterpret_cast<const int4*>(times)[i];
    uint32_t* bits_to = seen + (int64_t)slot * words + (first >> 5);
    if (t < min(kNotePart / 32, words - (first >> 5))) bits_to[t] = bits[t];
}

__device__ __forceinline__ void note(uint32_t* bits, int* times, int token, int vocab, bool counted) {
    if (token < 0 || token >= vocab) return;
    atomicOr(bits + (token >> 5), 1u << (token & 31));
    if (counted) atomicAdd(times + token, 1);
}

// grid: rows.  More of a row's tokens into its slot's history.
__global__ void __launch_bounds__(kNoteThreads)
note_kernel(uint32_t* __restrict__ seen, int* __restrict__ counts, int slot_count, int words, int stride, int vocab,
            const int* __restrict__ slots, const int* __restrict__ tokens, int total, const int* __restrict__ starts,
            const int* __restrict__ prompts) {
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x, slot = slots[row];
    if (slot < 0 || slot >= slot_count) return;
    const int begin = max(0, starts[row]), end = min(total, starts[row + 1]);
    const int prompt = prompts != nullptr ? prompts[row] : 0;
    for (int i = begin + (int)threadIdx.x; i < end; i += kNoteThreads)
        note(seen + (int64_t)slot * words, counts + (int64_t)slot * stride, tokens[i], vocab, i - begin >= prompt);
}

// A token a row: a decode step.
__global__ void __launch_bounds__(128)
note_one_kernel(uint32_t* __restrict__ seen, int* __restrict__ counts, int slot_count, int words, int stride, int vocab,
                const int* __restrict__ slots, const int* __restrict__ tokens, const int* __restrict__ prompts, int rows) {
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.x * 128 + threadIdx.x;
    if (row >= rows) return;
    const int slot = slots[row];
    if (slot < 0 || slot >= slot_count) return;
    note(seen + (int64_t)slot * words, counts + (int64_t)slot * stride, tokens[row], vocab, prompts == nullptr || prompts[row] <= 0);
}

// A slot's row of the table, which travels in the launch.
__global__ void set_kernel(SlotRules* to, SlotRules row) { *to = row; }

// ---- logits
//
// 8 V bytes a row are read and written (less where the mask rules out four neighbours: those are not read): 64 rows of 128,256 without
// rules take 13.5 us (4.9 TB/s), with a mask 15.7, with penalties, biases and a mask 23.6.  What bounds those is the blocks' own chain
// (slot, the slot's rules and its bits, behind which the logits are asked for; counts, 64-bit arithmetic between barriers: a third of all
// warps' time) with four blocks a multiprocessor; more blocks with fewer registers were no faster.  A block has 4,096 tokens, every so
// many-th run of 128 (low ids are had more often than high ones).  While its logits are on their way it lists the tokens that were had (a
// bit each), so that every thread has as many of them, and works those out in 64 bits; then everything is written, the listed ones
// behind the others.

constexpr int kShapeThreads = 256;
constexpr int kShapePart = 4096;
constexpr int kRun = 128;
constexpr int kEach = kShapePart / kShapeThreads;

// grid (parts of the vocabulary, rows).
__global__ void __launch_bounds__(kShapeThreads)
shape_kernel(const float* logits, int64_t stride, float* out, int64_t out_stride, int vocab, Rules rules) {
    __shared__ uint32_t mask[kShapePart / 32], had[kShapePart / 32];
    __shared__ uint16_t some[kShapePart];
    __shared__ float made[kShapePart];
    __shared__ int warps[kShapeThreads / 32];
    constexpr int kBiased = kMaxBiases / kShapeThreads;
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.y, t = threadIdx.x, lane = t & 31, warp = t >> 5, part = blockIdx.x, parts = gridDim.x;
    // the block's tokens are numbered 0 ... 4,095; which one of the vocabulary a number stands for
    auto token_of = [&](int i) { return ((i / kRun) * parts + part) * kRun + i % kRun; };
    const float* x = logits + (int64_t)row * stride;
    float* y = out + (int64_t)row * out_stride;
    const int slot = rules.slots[row];
    SlotRules rule = {};
    if (slot >= 0 && slot < rules.slot_count) rule = rules.table[slot];
    const bool masked = rule.kinds & kMask, penalised = rule.kinds & kPenalties;
    const int biases = rule.kinds & kBiases ? min(rule.biases, rules.room) : 0;
    const bool wide = (((uintptr_t)x | (uintptr_t)y) & 15) == 0;
    const bool in_place = x == y;
    if (in_place && rule.kinds == 0) return;
    if (t < kShapePart / 32) {
        const int token = token_of(32 * t), left = vocab - token;     // (of a word; what is behind the vocabulary is not allowed)
        const int64_t at = (int64_t)slot * rules.words + (token >> 5);
        const uint32_t there = left >= 32 ? ~0u : left > 0 ? ~0u >> (32 - left) : 0u;
        mask[t] = masked && left > 0 ? rules.masks[at] & there : there;
        had[t] = penalised && left > 0 ? rules.seen[at] & there : 0u;
    }
    __syncthreads();
    // ---- the logits: four neighbours where they are aligned, else one of every 256
    float v[kEach];
    auto place = [&](int u) { return wide ? (u >> 2) * 4 * kShapeThreads + 4 * t + (u & 3) : u * kShapeThreads + t; };
    auto allowed = [&](int i) { return mask[i >> 5] >> (i & 31) & 1; };
    if (!in_place || masked) {
        if (wide) {
#pragma unroll
            for (int u = 0; u < kEach; u += 4) {
                const int i = place(u), token = token_of(i);
                const bool any = mask[i >> 5] >> (i & 31) & 15;
                if (any && token + 4 <= vocab) {
                    const float4 four = *reinterpret_cast<const float4*>(x + token);
                    v[u] = four.x, v[u + 1] = four.y, v[u + 2] = four.z, v[u + 3] = four.w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[u + j] = any && token + j < vocab ? x[token + j] : -INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const int i = place(u);
                v[u] = allowed(i) ? x[token_of(i)] : -INFINITY;
            }
        }
    }
    // ---- the tokens that were had and those with a bias
    int listed = 0;
    if (penalised) {
        uint32_t bits = t < kShapePart / 32 ? had[t] : 0;
        const int mine = __popc(bits);
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += other;
        }
        if (lane == 31) warps[warp] = incl;
        __syncthreads();
        int at = incl - mine;
#pragma unroll
        for (int w = 0; w < kShapeThreads / 32; ++w) {
            if (w < warp) at += warps[w];
            listed += warps[w];
        }
        while (bits) {
            some[at++] = (uint16_t)(t * 32 + __ffs(bits) - 1);
            bits &= bits - 1;
        }
        __syncthreads();
        const int* counts = rules.counts + (int64_t)slot * rules.stride;
#pragma unroll 2
        for (int e = t; e < listed; e += kShapeThreads) {
            const int i = some[e];
            made[e] = allowed(i) ? shaped_logit(x[token_of(i)], rule, true, counts[token_of(i)], 0.0f) : -INFINITY;
        }
    }
    float biased[kBiased];
    auto mine = [&](int token) { return token >= 0 && token < vocab && token / kRun % parts == part; };
    if (biases > 0) {
        const int64_t at = (int64_t)slot * rules.room;
#pragma unroll
        for (int u = 0; u < kBiased; ++u) {
            const int e = t + u * kShapeThreads, token = e < biases ? rules.bias_ids[at + e] : -1;
            if (!mine(token)) continue;
            const int i = token / kRun / parts * kRun + token % kRun;
            const bool was = had[i >> 5] >> (i & 31) & 1;
            biased[u] = !allowed(i) ? -INFINITY
                                    : shaped_logit(x[token], rule, was, was ? rules.counts[(int64_t)slot * rules.stride + token] : 0,
                                                   rules.biases[at + e]);
        }
    }
    __syncthreads();                               // (in place: every logit that is needed has been read)
    if (!in_place || masked) {
        if (wide) {
#pragma unroll
            for (int u = 0; u < kEach; u += 4) {
                const int i = place(u), token = token_of(i);
                const uint32_t bits = mask[i >> 5] >> (i & 31);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[u + j] = bits >> j & 1 ? v[u + j] : -INFINITY;
                if (token + 4 <= vocab) {
                    *reinterpret_cast<float4*>(y + token) = make_float4(v[u], v[u + 1], v[u + 2], v[u + 3]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (token + j < vocab) y[token + j] = v[u + j];
                }
            }
        } else {
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const int token = token_of(place(u));
                if (token < vocab) y[token] = v[u];
            }
        }
    }
    if (penalised) {
        __syncthreads();
        for (int e = t; e < listed; e += kShapeThreads) y[token_of(some[e])] = made[e];
    }
    if (biases > 0) {
        __syncthreads();
        const int64_t at = (int64_t)slot * rules.room;
#pragma unroll
        for (int u = 0; u < kBiased; ++u) {
            const int e = t + u * kShapeThreads, token = e < biases ? rules.bias_ids[at + e] : -1;
            if (mine(token)) y[token] = biased[u];
        }
    }
}

}  // namespace

TB_EXPORT int tb_note_tokens(uint32_t* seen, int* counts, int slot_count, int words, int stride, int vocab, const int* slots,
                             const int* tokens, int total, const int* starts, const int* prompts, int rows, int restart,
                             cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0 || words < (vocab + 31) / 32 || stride < vocab || stride % 4 != 0) return TB_ERR_BAD_SIZE;
    if ((uintptr_t)counts & 15) return TB_ERR_BAD_ALIGN;
    cudaError_t err;
    if (restart) {
        if (rows > 65535) return TB_ERR_BAD_SIZE;
        err = tb_launch_pdl(restart_kernel, dim3((stride + kNotePart - 1) / kNotePart, rows), dim3(kNoteThreads), 0, stream, seen, counts,
                            slot_count, words, stride, vocab, slots, tokens, total, starts, prompts, rows);
    } else if (starts != nullptr) {
        err = tb_launch_pdl(note_kernel, dim3(rows), dim3(kNoteThreads), 0, stream, seen, counts, slot_count, words, stride, vocab, slots,
                            tokens, total, starts, prompts);
    } else {
        err = tb_launch_pdl(note_one_kernel, dim3((rows + 127) / 128), dim3(128), 0, stream, seen, counts, slot_count, words, stride, vocab,
                            slots, tokens, prompts, rows);
    }
    return err == cudaSuccess ? tb_launch_status() : (int)err;
}

TB_EXPORT int tb_set_rules(SlotRules* to, SlotRules row, cudaStream_t stream) {
    set_kernel<<<1, 1, 0, stream>>>(to, row);
    return tb_launch_status();
}

TB_EXPORT int tb_shape_logits(const float* logits, int64_t stride, float* out, int64_t out_stride, int rows, int vocab, Rules rules,
                              cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0 || rows > 65535 || rules.room > kMaxBiases) return TB_ERR_BAD_SIZE;
    const cudaError_t err = tb_launch_pdl(shape_kernel, dim3((vocab + kShapePart - 1) / kShapePart, rows), dim3(kShapeThreads), 0, stream,
                                          logits, stride, out, out_stride, vocab, rules);
    return err == cudaSuccess ? tb_launch_status() : (int)err;
}
