// One token a row from 32-bit logits: greedy, or drawn after top-k, min-p and top-p.
//
//   T <= 0: the lowest id of the largest logit.  Else, with z = x * (1 / T) and d = z - max z, each rounded to 32 bits (the
//   arithmetic of sample_top_p_host), weights w = e^d in 64 bits and tokens ranked by descending d, equal ones by id:
//     kept = the first top_k of the rank; of those w >= min_p; of those the shortest beginning with mass >= top_p * their mass
//     token = the first of the rank whose cumulative weight is above u * (mass of what is kept)
//   A row without any cut is drawn from in the order of ids with d = fma(x, 1 / T, -max z), as tb_sample does.
//   A row with NaN or +inf, or with nothing above -inf, has no token: -1.  Where 1 / T or a product with it leaves the 32 bits' range and
//   d is no number, the largest logits have d = 0 and the others -inf.
//
// What is kept is always a beginning of the rank: all tokens with d above some number, and the first j of those equal to it.  So every
// cut, and the draw itself, asks for the place in the rank where a cumulative measure (a count or a mass) first reaches a number.
#include "common.cuh"

namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ uint32_t ordered(float v) {       // floats as unsigned numbers of the same order
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

template <typename T, typename Op>
__device__ T block_reduce(T v, T* scratch, Op op) {
    for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    T all = scratch[0];
    for (int w = 1; w < kWarps; ++w) all = op(all, scratch[w]);
    return all;
}

struct Place {          // a beginning of the rank: everything with d above `d`, and the first `equals` (by id) of those equal to it
    float d;
    int equals;
    double mass;        // its measure
};

struct Row {
    const float* x;
    int vocab;
    float inverse, best, top;
    __device__ float number(float l, float d) const { return d == d ? d : l == best ? 0.0f : -INFINITY; }
    __device__ float distance(int i) const { return number(x[i], __fsub_rn(__fmul_rn(x[i], inverse), top)); }
    __device__ float distance_once(int i) const { return number(x[i], fmaf(x[i], inverse, -top)); }
};

// The first place of the rank, within `bound`, whose cumulative measure is at least (`above`: more than) `target`.
__device__ Place locate(const Row& row, bool mass, double target, bool above, const Place& bound, double* scratch) {
    auto sum = [](double a, double b) { return a + b; };
    const double last = mass ? exp((double)bound.d) : 1.0;
    auto reach = [&](double v) { return above ? v > target : v >= target; };
    auto measure = [&](float from, bool open) {              // of what is in the bound with d >= from (open: d > from)
        double mine = 0.0;
        for (int i = threadIdx.x; i < row.vocab; i += kThreads) {
            const float d = row.distance(i);
            if ((open ? d > from : d >= from) && d > bound.d) mine += mass ? exp((double)d) : 1.0;
        }
        mine = block_reduce(mine, scratch, sum);
        return (open ? from < bound.d : from <= bound.d) ? mine + (double)bound.equals * last : mine;
    };
    if (!reach(measure(bound.d, false))) return bound;
    uint32_t low = ordered(bound.d), high = ordered(0.0f) + 1;       // reached from `low` on, not from `high`
    while (high > low + 1) {
        const uint32_t middle = low + (high - low) / 2;
        if (reach(measure(from_ordered(middle), false))) low = middle; else high = middle;
    }
    Place place;
    place.d = from_ordered(low);
    const double in_front = measure(place.d, true), each = mass ? exp((double)place.d) : 1.0;
    int equals = 0;
    for (int i = threadIdx.x; i < row.vocab; i += kThreads) equals += row.distance(i) == place.d;
    equals = (int)block_reduce((double)equals, scratch, sum);
    if (place.d == bound.d) equals = min(equals, bound.equals);
    int first = 1;
    for (int step = 1 << 30; step > 0; step >>= 1)           // the fewest that reach it
        if (first + step <= equals && !reach(in_front + (double)(first + step - 1) * each)) first += step;
    place.equals = first;
    place.mass = in_front + (double)first * each;
    return place;
}

__global__ void __launch_bounds__(kThreads)
choose_kernel(const float* __restrict__ logits, int64_t stride, const float* __restrict__ temperature, const double* __restrict__ uniform,
              const int* __restrict__ top_k, const double* __restrict__ top_p, const double* __restrict__ min_p,
              int* __restrict__ out, int vocab) {
    __shared__ double scratch[kWarps];
    __shared__ int picked;
    const int r = blockIdx.x;
    const float* x = logits + (int64_t)r * stride;
    const float t = temperature[r];
    auto most = [](float a, float b) { return fmaxf(a, b); };
    float best = -INFINITY;
    int broken = 0;
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
        best = fmaxf(best, x[i]);
        broken |= !(x[i] < INFINITY);
    }
    best = block_reduce(best, reinterpret_cast<float*>(scratch), most);
    broken = __syncthreads_or(broken);
    if (broken || best == -INFINITY) {
        if (threadIdx.x == 0) out[r] = -1;
        return;
    }
    if (threadIdx.x == 0) picked = vocab;
    __syncthreads();
    if (!(t > 0.0f)) {
        for (int i = threadIdx.x; i < vocab; i += kThreads)
            if (x[i] == best) {
                atomicMin(&picked, i);
                break;
            }
        __syncthreads();
        if (threadIdx.x == 0) out[r] = picked;
        return;
    }
    const int k = top_k != nullptr ? top_k[r] : 0;
    const double p = top_p != nullptr ? top_p[r] : 1.0, floor = min_p != nullptr ? min_p[r] : 0.0, u = uniform[r];
    const Row row = {x, vocab, 1.0f / t, best, best * (1.0f / t)};
    if (!((k > 0 && k < vocab) || p < 1.0 || floor > 0.0)) {
        // in the order of ids: a thread's part is a run of tokens
        const int part = (vocab + kThreads - 1) / kThreads, begin = min(vocab, (int)threadIdx.x * part), end = min(vocab, begin + part);
        auto weight = [&](int i) { return exp((double)row.distance_once(i)); };
        __shared__ double masses[kThreads];
        double mine = 0.0;
        for (int i = begin; i < end; ++i) mine += weight(i);
        masses[threadIdx.x] = mine;
        __syncthreads();
        if (threadIdx.x == 0) {
            double all = 0.0, run = 0.0;
            for (int i = 0; i < kThreads; ++i) all += masses[i];
            int token = -1;
            for (int i = 0; i < kThreads && token < 0; ++i) {
                if (run + masses[i] > u * all || i == kThreads - 1)
                    for (int j = min(vocab, i * part); j < min(vocab, i * part + part) && token < 0; ++j) {
                        run += weight(j);
                        if (run > u * all) token = j;
                    }
                else
                    run += masses[i];
            }
            out[r] = token < 0 ? vocab - 1 : token;
        }
        return;
    }
    Place kept = {-INFINITY, 0, 0.0};
    if (k > 0 && k < vocab) kept = locate(row, false, (double)k, false, kept, scratch);
    if (floor > 0.0) {
        const float from = __double2float_ru(log(floor));
        if (from > kept.d) kept = {from, 0x3fffffff, 0.0};
    }
    if (kept.d > 0.0f) kept.d = 0.0f;                        // (min_p above 1 keeps the largest)
    {
        // the mass of what is left, with no more equals than there are
        int equals = 0;
        for (int i = threadIdx.x; i < vocab; i += kThreads) equals += row.distance(i) == kept.d;
        equals = (int)block_reduce((double)equals, scratch, [](double a, double b) { return a + b; });
        kept.equals = min(kept.equals, equals);
        double mine = 0.0;
        for (int i = threadIdx.x; i < vocab; i += kThreads) {
            const float d = row.distance(i);
            if (d > kept.d) mine += exp((double)d);
        }
        kept.mass = block_reduce(mine, scratch, [](double a, double b) { return a + b; }) + kept.equals * exp((double)kept.d);
    }
    if (p < 1.0) kept = locate(row, true, kept.mass * p, false, kept, scratch);
    const Place drawn = locate(row, true, kept.mass * u, true, kept, scratch);
    // the drawn.equals-th by id of those at drawn.d
    if (threadIdx.x < 32) {
        int left = drawn.equals, token = vocab - 1;
        for (int base = 0; base < vocab; base += 32) {
            const int i = base + (int)threadIdx.x;
            unsigned here = __ballot_sync(0xffffffffu, i < vocab && row.distance(i) == drawn.d);
            const int n = __popc(here);
            if (n >= left) {
                for (; left > 1; --left) here &= here - 1;
                token = base + __ffs(here) - 1;
                break;
            }
            left -= n;
        }
        if (threadIdx.x == 0) out[r] = token;
    }
}

}  // namespace

TB_EXPORT int tb_choose_tokens(const float* logits, int64_t stride, const float* temperature, const double* uniform, const int* top_k,
                               const double* top_p, const double* min_p, int* out, int rows, int vocab, cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0) return TB_ERR_BAD_SIZE;
    choose_kernel<<<rows, kThreads, 0, stream>>>(logits, stride, temperature, uniform, top_k, top_p, min_p, out, vocab);
    return tb_launch_status();
}
