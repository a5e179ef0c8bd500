// Histories of tokens a request, and logits under a request's rules (token_rules.cuh).
#include "token_rules.cuh"

namespace {

constexpr int kThreads = 1024;

// grid: rows.  A row's known tokens into its slot's history; `restart`: in place of what stands there (then of rows that name one
// slot the last counts).
__global__ void __launch_bounds__(kThreads)
note_kernel(uint32_t* __restrict__ seen, int* __restrict__ counts, int slot_count, int words, int stride, int vocab,
            const int* __restrict__ slots, const int* __restrict__ tokens, int total, const int* __restrict__ starts,
            const int* __restrict__ prompts, int rows, int restart) {
    const int row = blockIdx.x, slot = slots[row];
    if (slot < 0 || slot >= slot_count) return;
    uint32_t* bits = seen + (int64_t)slot * words;
    int* times = counts + (int64_t)slot * stride;
    if (restart) {
        int later = 0;
        for (int r = row + 1 + threadIdx.x; r < rows; r += kThreads) later |= slots[r] == slot;
        if (__syncthreads_or(later)) return;
        for (int i = threadIdx.x; i < words; i += kThreads) bits[i] = 0;
        for (int i = threadIdx.x; i < stride; i += kThreads) times[i] = 0;
        __syncthreads();
    }
    const int begin = starts != nullptr ? max(0, starts[row]) : row;
    const int end = starts != nullptr ? min(total, starts[row + 1]) : row + 1;
    const int prompt = prompts != nullptr ? prompts[row] : 0;
    for (int i = begin + (int)threadIdx.x; i < end; i += kThreads) {
        const int token = tokens[i];
        if (token < 0 || token >= vocab) continue;
        atomicOr(bits + (token >> 5), 1u << (token & 31));
        if (i - begin >= prompt) atomicAdd(times + token, 1);
    }
}

// grid: rows.
__global__ void __launch_bounds__(kThreads)
shape_kernel(const float* logits, int64_t stride, float* out, int64_t out_stride, int vocab, Rules rules) {
    __shared__ float raw[kMaxBiases];
    const int row = blockIdx.x;
    const float* x = logits + (int64_t)row * stride;
    float* y = out + (int64_t)row * out_stride;
    const int slot = rules.slots[row];
    SlotRules rule = {};
    if (slot >= 0 && slot < rules.slot_count) rule = rules.table[slot];
    const uint32_t* seen = rules.seen + (int64_t)slot * rules.words;
    const uint32_t* mask = rules.masks + (int64_t)slot * rules.words;
    const int* counts = rules.counts + (int64_t)slot * rules.stride;
    const int* ids = rules.bias_ids + (int64_t)slot * rules.room;
    const int biases = rule.kinds & kBiases ? min(rule.biases, rules.room) : 0;
    for (int i = threadIdx.x; i < biases; i += kThreads) {
        const int token = ids[i];
        raw[i] = token >= 0 && token < vocab ? x[token] : 0.0f;
    }
    __syncthreads();
    auto shaped = [&](int token, float l, float bias) {
        if (rule.kinds & kMask && !(mask[token >> 5] >> (token & 31) & 1)) return -INFINITY;
        const bool had = rule.kinds & kPenalties && seen[token >> 5] >> (token & 31) & 1;
        if (!had && bias == 0.0f) return l;
        return shaped_logit(l, rule, had, had ? counts[token] : 0, bias);
    };
    for (int i = threadIdx.x; i < vocab; i += kThreads) y[i] = shaped(i, x[i], 0.0f);
    __syncthreads();
    for (int i = threadIdx.x; i < biases; i += kThreads) {
        const int token = ids[i];
        if (token >= 0 && token < vocab) y[token] = shaped(token, raw[i], rules.biases[(int64_t)slot * rules.room + i]);
    }
}

}  // namespace

TB_EXPORT int tb_note_tokens(uint32_t* seen, int* counts, int slot_count, int words, int stride, int vocab, const int* slots,
                             const int* tokens, int total, const int* starts, const int* prompts, int rows, int restart,
                             cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0 || words < (vocab + 31) / 32 || stride < vocab) return TB_ERR_BAD_SIZE;
    note_kernel<<<rows, kThreads, 0, stream>>>(seen, counts, slot_count, words, stride, vocab, slots, tokens, total, starts, prompts,
                                               rows, restart);
    return tb_launch_status();
}

TB_EXPORT int tb_shape_logits(const float* logits, int64_t stride, float* out, int64_t out_stride, int rows, int vocab, Rules rules,
                              cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0 || rules.room > kMaxBiases) return TB_ERR_BAD_SIZE;
    shape_kernel<<<rows, kThreads, 0, stream>>>(logits, stride, out, out_stride, vocab, rules);
    return tb_launch_status();
}
