// One token a row from 32-bit logits under the row's rules (token_rules.cuh): greedy, or drawn after top-k, min-p and top-p.
//
//   T <= 0: the lowest id of the largest logit.  Else, with z = x * (1 / T) and d = z - max z, each rounded to 32 bits (the
//   arithmetic of sample_top_p_host), weights w = e^d in 64 bits and tokens ranked by descending d, equal ones by id:
//     kept = the first top_k of the rank; of those w >= min_p; of those the shortest beginning with mass >= top_p * their mass
//     token = the first of the rank whose cumulative weight is above u * (mass of what is kept)
//   A row without any cut is drawn from in the order of ids with d = fma(x, 1 / T, -max z), as tb_sample does (where max z is 65,536 and
//   more, at temperatures of a thousandth and below, that would leave the largest logit itself away from 0: there d as above).
//   A row with NaN or +inf, or with nothing above -inf, has no token: -1.  Where max z leaves the 32 bits' range, the largest logits have
//   d = 0 and the others -inf.
//
// A row is shared by a thread-block cluster; each block reads its part of the vocabulary once, into shared memory, and all that follows
// runs there.  The tokens are counted in 1,024 bins of d.  The counts say how far down the rank a cut can reach at most (of a bin's
// tokens none weighs less than its lower edge), and where that is no more than kListed tokens, which nearly all calls are, they
// are listed, one block sorts them, and sums of their weights in the order of the rank give every cut and the token.  Otherwise
// each cut, and then the draw, is looked for by itself: sums over the bins that are certainly in front of it, a list of those that it may
// lie in.  Where even those are more than a list holds (great numbers of equal logits), the interval of d is halved.
#include "token_rules.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 8;
constexpr int kMaxChunk = 32768;         // tokens of a block
constexpr int kBins = 1024;
constexpr int kListed = 2048;
constexpr int kTable = 32;
constexpr float kReach = 32.0f;          // the bins cover d down to -32 at most; what is below is in the last
constexpr double kSpare = 1e-5;          // of a mass bound by a bin's edges: d * scale is within 2^-23 of it, e^-32 of e^(-32 (1 + 2^-23)) within 4e-6
constexpr uint64_t kLast = ~0ull;

struct Shared {
    alignas(16) uint32_t hist[kBins];    // first the mask's words (32 tokens each), then counts a bin
    double table[kTable];                // 2^(i / 32)
    double sums[kWarps];
    int counts[kWarps];
    int listed;
    int edge, before;
    double answer;
    // what the other blocks of the cluster read
    float best, low;
    int broken, first;
    double mass[2];
    int total[2];
    uint64_t place;
    double place_sum;
};

__device__ __forceinline__ uint32_t peer_address(const void* local, uint32_t rank) {
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    return remote;
}
__device__ __forceinline__ uint32_t peer_u32(const void* local, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(peer_address(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint64_t peer_u64(const void* local, uint32_t rank) {
    uint64_t v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(peer_address(local, rank)) : "memory");
    return v;
}
__device__ __forceinline__ int peer(const int* local, uint32_t rank) { return (int)peer_u32(local, rank); }
__device__ __forceinline__ float peer(const float* local, uint32_t rank) { return __uint_as_float(peer_u32(local, rank)); }
__device__ __forceinline__ double peer(const double* local, uint32_t rank) { return __longlong_as_double((long long)peer_u64(local, rank)); }

__device__ __forceinline__ void copy16(uint32_t to, const float* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }

// e^d for d <= 0 (and -inf) in 64 bits, by a table of 2^(i / 32) and a polynomial of what is left (P. T. P. Tang, "Table-driven
// implementation of the exponential function in IEEE floating-point arithmetic", 1989): d = (32 m + i) ln 2 / 32 + r with |r| <= ln 2 / 64,
// e^r by its series up to r^5 (the rest is below 3e-15).  With the rounding of d's reduction the relative error is below 1e-14 + 1e-16 |d|.
__device__ __forceinline__ double weight_of(float d, const double* table) {
    if (!(d > -700.0f)) return 0.0;      // (below 10^-304: nothing beside the largest weight, which is 1)
    constexpr double kSteps = 32.0 / 0.693147180559945309417232121458, kStep = 0.693147180559945309417232121458 / 32.0;
    constexpr double kRound = 6755399441055744.0;                              // 1.5 * 2^52: adding it rounds to a whole number
    const double x = (double)d, whole = fma(x, kSteps, kRound);
    const int n = __double2loint(whole);
    const double r = fma(whole - kRound, -kStep, x);
    const double series = fma(r, fma(r, fma(r, fma(r, fma(r, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0);
    return table[n & (kTable - 1)] * series * __hiloint2double((1023 + (n >> 5)) << 20, 0);
}

// A token's place in the rank: ascending keys.
__device__ __forceinline__ uint64_t key_of(float d, int id) { return (uint64_t)__float_as_uint(fabsf(d)) << 32 | (uint32_t)id; }
__device__ __forceinline__ float distance_of(uint64_t key) { return -__uint_as_float((uint32_t)(key >> 32)); }

struct Row {
    Shared& sh;
    float* s;                            // the block's tokens: logits, later distances
    uint64_t* list;
    int first, count;                    // its tokens: ids first ... first + count - 1
    int block, blocks, turn;
    float scale;                         // bins a unit of d

    __device__ __forceinline__ int lane() const { return threadIdx.x & 31; }
    __device__ __forceinline__ int warp() const { return threadIdx.x >> 5; }
    __device__ __forceinline__ void meet() const {                     // all threads of the cluster
        if (blocks > 1)
            asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        else
            __syncthreads();
    }
    __device__ __forceinline__ int bin(float d) const {
        const float at = -d * scale;
        return at < (float)(kBins - 1) ? (int)at : kBins - 1;
    }

    // ---- sums, in a fixed order
    __device__ double block_sum(double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if (lane() == 0) sh.sums[warp()] = v;
        __syncthreads();
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all += sh.sums[w];
        return all;
    }
    __device__ int block_count(int v) {
        v = __reduce_add_sync(0xffffffffu, v);
        __syncthreads();
        if (lane() == 0) sh.counts[warp()] = v;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) all += sh.counts[w];
        return all;
    }
    // (two places in turn: whoever writes one again has passed a barrier behind everyone's reading of it)
    __device__ double row_sum(double v) {
        v = block_sum(v);
        if (blocks == 1) return v;
        if (threadIdx.x == 0) sh.mass[turn] = v;
        meet();
        double all = 0.0;
        for (int b = 0; b < blocks; ++b) all += peer(&sh.mass[turn], b);
        turn ^= 1;
        return all;
    }
    __device__ int row_count(int v) {
        v = block_count(v);
        if (blocks == 1) return v;
        if (threadIdx.x == 0) sh.total[turn] = v;
        meet();
        int all = 0;
        for (int b = 0; b < blocks; ++b) all += peer(&sh.total[turn], b);
        turn ^= 1;
        return all;
    }
    template <typename T>
    __device__ T sum_before(T mine, T* scratch) {                      // exclusive, over the block's threads in order
        T incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T other = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane() >= o) incl += other;
        }
        __syncthreads();
        if (lane() == 31) scratch[warp()] = incl;
        __syncthreads();
        T before = 0;
        for (int w = 0; w < kWarps; ++w)
            if (w < warp()) before += scratch[w];
        T own = __shfl_up_sync(0xffffffffu, incl, 1);
        return before + (lane() == 0 ? (T)0 : own);
    }

    // ---- the list: the block's tokens in bins from ... to that rank no later than `bound`; then the whole row's in the first block
    // Returns where the row's entries are (first block) and how many.  Every block must know that they fit.
    template <typename Keep>
    __device__ uint64_t* gather(Keep keep, int& n) {
        if (threadIdx.x == 0) sh.listed = 0;
        uint64_t mine = 0;                                             // a bit a token of the thread's
        for (int i = threadIdx.x, at = 0; i < count; i += kThreads, ++at)
            if (keep(s[i], first + i)) mine |= 1ull << at;
        const int here = __popcll(mine);
        int incl = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane() >= o) incl += other;
        }
        __syncthreads();
        int base = 0;
        if (lane() == 31 && incl > 0) base = atomicAdd(&sh.listed, incl);      // (any order: the list is sorted)
        int at = __shfl_sync(0xffffffffu, base, 31) + incl - here;
        while (mine) {
            const int i = threadIdx.x + (__ffsll((long long)mine) - 1) * kThreads;
            mine &= mine - 1;
            list[at++] = key_of(s[i], first + i);
        }
        meet();
        n = sh.listed;
        if (blocks == 1) return list;
        uint64_t* all = reinterpret_cast<uint64_t*>(s);
        return all;
    }
    // (the first block takes the others' entries over the place of `s`, or behind its own)
    __device__ void pull(uint64_t* to, int& n) {
        int at = 0;
        for (int b = 0; b < blocks; ++b) {
            const int theirs = peer(&sh.listed, b);
            for (int e = threadIdx.x; e < theirs; e += kThreads) to[at + e] = peer_u64(list + e, b);
            at += theirs;
        }
        n = at;
        __syncthreads();
    }

    // ascending; `n` entries, room for the next power of two
    __device__ void sort(uint64_t* keys, int n) {
        int size = 64;
        while (size < n) size <<= 1;
        for (int i = n + (int)threadIdx.x; i < size; i += kThreads) keys[i] = kLast;
        __syncthreads();
        for (int run = 2; run <= size; run <<= 1)
            for (int step = run >> 1; step > 0; step >>= 1) {
                // (up to 32 apart a warp's pairs lie within 64 entries of its own)
                for (int p = threadIdx.x; p < size >> 1; p += kThreads) {
                    const int i = 2 * p - (p & (step - 1)), j = i + step;
                    const uint64_t a = keys[i], b = keys[j];
                    if ((a > b) == ((i & run) == 0)) {
                        keys[i] = b;
                        keys[j] = a;
                    }
                }
                if (step > 32 || (step == 1 && run >= 64)) __syncthreads(); else __syncwarp();
            }
        __syncthreads();
    }
};

// Sums over a sorted list of the weights of its first `n` entries; every thread has a run of entries.
struct Ranked {
    Row& row;
    const uint64_t* keys;
    int each, begin, end;
    double before;                       // in front of the thread's

    __device__ Ranked(Row& row, const uint64_t* keys, int n) : row(row), keys(keys) {
        each = (n + kThreads - 1) / kThreads;
        begin = min(n, (int)threadIdx.x * each);
        end = min(n, begin + each);
        double mine = 0.0;
        for (int e = begin; e < end; ++e) mine += weight_of(distance_of(keys[e]), row.sh.table);
        before = row.sum_before(mine, row.sh.sums);
    }
    // How many entries' cumulative sums do not reach `target` (`above`: are not above it).
    __device__ int short_of(double target, bool above, double base) {
        double run = base + before;
        int mine = 0;
        for (int e = begin; e < end; ++e) {
            run += weight_of(distance_of(keys[e]), row.sh.table);
            if (above ? run > target : run >= target) break;
            ++mine;
        }
        return row.block_count(mine);
    }
    __device__ double sum_through(int place) {                          // of the entries up to and with `place`
        if (place >= begin && place < end) {
            double run = before;
            for (int e = begin; e <= place; ++e) run += weight_of(distance_of(keys[e]), row.sh.table);
            row.sh.answer = run;
        }
        __syncthreads();
        const double sum = row.sh.answer;
        __syncthreads();
        return sum;
    }
};

// The first token of the rank, within `bound`, at which a cumulative measure (its mass, or a count) reaches `target` (`above`: is above
// it), when more tokens than a list holds come into question; they lie in [low, high].  Every block has the same answer.
__device__ uint64_t halve(Row& row, bool mass, double target, bool above, uint64_t low, uint64_t high, double& sum) {
    constexpr int kIds = 18;                                            // (bits of an id: kMaxBlocks * kMaxChunk tokens)
    auto reach = [&](double v) { return above ? v > target : v >= target; };
    auto narrow = [&](uint64_t key) { return key >> 32 << kIds | min((unsigned long long)((1 << kIds) - 1), (unsigned long long)(key & 0xffffffffull)); };
    auto upto = [&](uint64_t place) {
        double mine = 0.0;
        for (int i = threadIdx.x; i < row.count; i += kThreads) {
            const float d = row.s[i];
            if (d > -INFINITY && narrow(key_of(d, row.first + i)) <= place) mine += mass ? weight_of(d, row.sh.table) : 1.0;
        }
        return row.row_sum(mine);
    };
    low = narrow(low);
    high = narrow(high);
    sum = upto(high);
    if (!reach(sum)) {                                                  // (rounding, or fewer tokens than asked for: the last one)
        target = sum;
        above = false;
    }
    while (low < high) {
        const uint64_t middle = low + (high - low) / 2;
        const double v = upto(middle);
        if (reach(v)) {
            high = middle;
            sum = v;
        } else {
            low = middle + 1;
        }
    }
    return high >> kIds << 32 | (high & ((1 << kIds) - 1));
}

// The same by the bins: `cumulative` are the tokens up to and with a bin (this thread's two bins: 2 t and 2 t + 1).
struct Bins {
    int own[2], cumulative[2];
    double least[2], most[2];            // bounds of the mass up to and with a bin
};

__device__ uint64_t locate(Row& row, const Bins& bins, bool mass, double target, bool above, uint64_t bound, double& sum) {
    Shared& sh = row.sh;
    // the bins that it may lie in
    int from = kBins, to = kBins;
    for (int e = 1; e >= 0; --e) {
        const int b = 2 * threadIdx.x + e;
        // (a millionth to spare for the bounds' own rounding and that of a bin's edges)
        const double low = mass ? bins.least[e] * (1.0 - kSpare) : (double)bins.cumulative[e];
        const double high = mass ? bins.most[e] * (1.0 + kSpare) : (double)bins.cumulative[e];
        if (high >= target) from = b;
        if (above ? low > target : low >= target) to = b;
    }
    const int last = bound == kLast ? kBins - 1 : row.bin(distance_of(bound));
    from = min(__reduce_min_sync(0xffffffffu, from), last);
    to = min(__reduce_min_sync(0xffffffffu, to), last);
    __syncthreads();
    if (threadIdx.x == 0) sh.edge = sh.before = kBins;
    __syncthreads();
    if (row.lane() == 0) {
        atomicMin(&sh.edge, from);
        atomicMin(&sh.before, to);
    }
    __syncthreads();
    from = min(sh.edge, last);
    to = min(sh.before, last);
    // tokens in front of the bins and in them
    int in_front = 0, through = 0;
    for (int e = 0; e < 2; ++e) {
        const int b = 2 * threadIdx.x + e;
        in_front += b < from ? bins.own[e] : 0;
        through += b <= to ? bins.own[e] : 0;
    }
    in_front = row.block_count(in_front);
    through = row.block_count(through);
    if (through - in_front > kListed) {
        const float unit = row.scale > 0.0f ? 1.0f / row.scale : 0.0f;
        return halve(row, mass, target, above, key_of((float)from * unit * (1.0f - (float)kSpare), 0),
                     to < kBins - 1 && row.scale > 0.0f ? (uint64_t)min((unsigned long long)bound, (unsigned long long)key_of((float)(to + 1) * unit * (1.0f + (float)kSpare), 0x7fffffff)) : bound,
                     sum);
    }
    double base = (double)in_front;
    if (mass) {
        double mine = 0.0;
        for (int i = threadIdx.x; i < row.count; i += kThreads) {
            const float d = row.s[i];
            if (d > -INFINITY && row.bin(d) < from) mine += weight_of(d, sh.table);
        }
        base = row.row_sum(mine);
    }
    int n;
    row.gather([&](float d, int id) {
        if (!(d > -INFINITY)) return false;
        const int b = row.bin(d);
        return b >= from && b <= to && key_of(d, id) <= bound;
    }, n);
    if (row.block == 0) {
        // (behind the block's own list there is room for a whole one)
        uint64_t* keys = row.blocks == 1 ? row.list : row.list + kListed;
        if (row.blocks > 1) row.pull(keys, n);
        row.sort(keys, n);
        int place;
        double through_place;
        if (mass) {
            Ranked ranked(row, keys, n);
            place = min(ranked.short_of(target, above, base), n - 1);
            through_place = base + (n > 0 ? ranked.sum_through(place) : 0.0);
        } else {
            place = min(max((int)(target - base) - 1, 0), n - 1);
            through_place = base + place + 1;
        }
        if (threadIdx.x == 0) {
            sh.place = n > 0 ? keys[place] : bound;
            sh.place_sum = through_place;
        }
    }
    row.meet();
    const uint64_t found = row.blocks > 1 ? peer_u64(&sh.place, 0) : sh.place;
    sum = row.blocks > 1 ? peer(&sh.place_sum, 0) : sh.place_sum;
    row.meet();                                                         // (the first block may write its answer again)
    return found;
}

// grid (blocks a row, rows); the blocks of a row are one cluster.
__global__ void __launch_bounds__(kThreads, 2)
choose_kernel(const float* __restrict__ logits, int64_t stride, const float* __restrict__ temperature, const double* __restrict__ uniform,
              const int* __restrict__ top_k, const double* __restrict__ top_p, const double* __restrict__ min_p, int* __restrict__ out,
              int vocab, int chunk, Rules rules) {
    __shared__ Shared sh;
    extern __shared__ uint4 dynamic[];
    pdl_trigger();
    pdl_wait();                                    // the logits, and the histories, come from kernels in front
    const int r = blockIdx.y, blocks = gridDim.x, block = blockIdx.x, t = threadIdx.x;
    const int first = min(vocab, block * chunk), count = min(vocab, first + chunk) - first;
    // ---- the block's tokens into shared memory; their first lies where 16-byte copies keep their alignment
    const float* x = logits + (int64_t)r * stride + first;
    const int shift = (int)((uintptr_t)x >> 2 & 3);
    uint64_t* list = reinterpret_cast<uint64_t*>(dynamic);
    float* s = reinterpret_cast<float*>(list + (blocks == 1 ? kListed : 2 * kListed)) + shift;
    const uint32_t s_at = (uint32_t)__cvta_generic_to_shared(s);
    {
        const int head = min(count, (4 - shift) & 3), packets = (count - head) >> 2;
        for (int p = t; p < packets; p += kThreads) copy16(s_at + 4 * (head + 4 * p), x + head + 4 * p);
        if (t < head) copy4(s_at + 4 * t, x + t);
        const int tail = head + 4 * packets + t;
        if (tail < count) copy4(s_at + 4 * tail, x + tail);
    }
    const int slot = rules.slots != nullptr ? rules.slots[r] : -1;
    SlotRules rule = {};
    if (slot >= 0 && slot < rules.slot_count) rule = rules.table[slot];
    const int words = (count + 31) >> 5;           // (a block begins with a word of its own)
    if (rule.kinds & kMask) {
        const uint32_t* mask = rules.masks + (int64_t)slot * rules.words + (first >> 5);
        const uint32_t hist_at = (uint32_t)__cvta_generic_to_shared(sh.hist);
        for (int w = t; w < words; w += kThreads) copy4(hist_at + 4 * w, mask + w);
    }
    const float temp = temperature[r];
    Row row = {sh, s, list, first, count, block, blocks, 0, 0.0f};
    // ---- penalties and biases, token by token
    if (rule.kinds & (kPenalties | kBiases)) {
        const uint32_t* seen = rules.seen + (int64_t)slot * rules.words + (first >> 5);
        const int* had = rules.counts + (int64_t)slot * rules.stride + first;
        const int biases = rule.kinds & kBiases ? min(rule.biases, rules.room) : 0;
        const int* ids = rules.bias_ids + (int64_t)slot * rules.room;
        constexpr int kMine = kMaxBiases / kThreads;
        float raw[kMine];
        copies_done();
        __syncthreads();
        for (int e = 0; e < kMine; ++e) {
            const int at = t + e * kThreads, i = at < biases ? ids[at] - first : -1;
            raw[e] = i >= 0 && i < count ? s[i] : 0.0f;
        }
        if (rule.kinds & kPenalties) {
            // the tokens that were had are listed, so that every thread has as many
            uint16_t* some = reinterpret_cast<uint16_t*>(list);
            for (int w0 = 0; w0 < words; w0 += kThreads) {
                uint32_t bits = w0 + t < words ? seen[w0 + t] : 0;
                if ((w0 + t) * 32 + 32 > count && w0 + t < words) bits &= ~0u >> (32 - (count - (w0 + t) * 32));
                const int mine = __popc(bits);
                int at = row.sum_before(mine, sh.counts);
                if (t == kThreads - 1) sh.listed = at + mine;
                while (bits) {
                    some[at++] = (uint16_t)((w0 + t) * 32 + __ffs(bits) - 1);
                    bits &= bits - 1;
                }
                __syncthreads();
                const int n = sh.listed;
                for (int e = t; e < n; e += kThreads) {
                    const int i = some[e];
                    s[i] = shaped_logit(s[i], rule, true, had[i], 0.0f);
                }
                __syncthreads();
            }
        }
        __syncthreads();
        for (int e = 0; e < kMine; ++e) {
            const int at = t + e * kThreads, i = at < biases ? ids[at] - first : -1;
            if (i < 0 || i >= count) continue;
            const bool was = rule.kinds & kPenalties && seen[i >> 5] >> (i & 31) & 1;
            s[i] = shaped_logit(raw[e], rule, was, was ? had[i] : 0, rules.biases[(int64_t)slot * rules.room + at]);
        }
    }
    if (t < kTable) sh.table[t] = exp2((double)t / kTable);
    copies_done();
    __syncthreads();
    // ---- the mask; the row's largest and smallest logit
    float best = -INFINITY, low = INFINITY;
    int broken = 0, lowest = 0x7fffffff;
    for (int i = t; i < count; i += kThreads) {
        float v = s[i];
        if (rule.kinds & kMask && !(sh.hist[i >> 5] >> (i & 31) & 1)) s[i] = v = -INFINITY;
        broken |= !(v < INFINITY);
        if (v > best) {
            best = v;
            lowest = first + i;
        }
        if (v > -INFINITY) low = fminf(low, v);
    }
    {
        const float mine = best;
        best = warp_max(best);
        lowest = (int)__reduce_min_sync(0xffffffffu, (unsigned)(mine == best ? lowest : 0x7fffffff));
        low = -warp_max(-low);
        broken = __any_sync(0xffffffffu, broken);
        float* scratch = reinterpret_cast<float*>(sh.sums);            // best, low a warp
        if (row.lane() == 0) {
            scratch[2 * row.warp()] = best;
            scratch[2 * row.warp() + 1] = low;
            sh.counts[row.warp()] = broken ? -1 : lowest;
        }
        __syncthreads();
        best = -INFINITY, low = INFINITY, broken = 0, lowest = 0x7fffffff;
        for (int w = 0; w < kWarps; ++w) {
            const float b = scratch[2 * w];
            const int l = sh.counts[w];
            broken |= l < 0;
            if (b > best || (b == best && l < lowest)) lowest = l;
            best = fmaxf(best, b);
            low = fminf(low, scratch[2 * w + 1]);
        }
        if (blocks > 1) {
            if (t == 0) {
                sh.best = best;
                sh.low = low;
                sh.first = broken ? -1 : lowest;
            }
            row.meet();
            best = -INFINITY, low = INFINITY, broken = 0, lowest = 0x7fffffff;
            for (int b = 0; b < blocks; ++b) {
                const float v = peer(&sh.best, b);
                const int l = peer(&sh.first, b);
                broken |= l < 0;
                if (v > best || (v == best && l < lowest)) lowest = l;
                best = fmaxf(best, v);
                low = fminf(low, peer(&sh.low, b));
            }
        }
    }
    if (broken || best == -INFINITY || !(temp > 0.0f)) {
        if (block == 0 && t == 0) out[r] = broken || best == -INFINITY ? -1 : lowest;
        row.meet();                                // no block leaves while a peer may still read its shared memory
        return;
    }
    const int k = top_k != nullptr ? top_k[r] : 0;
    const double p = top_p != nullptr ? top_p[r] : 1.0, floor = min_p != nullptr ? min_p[r] : 0.0, u = uniform[r];
    const float inverse = 1.0f / temp, top = best * inverse;
    const bool finite = fabsf(top) < INFINITY;
    auto number = [&](float l, float d) { return finite ? d : l == best ? 0.0f : -INFINITY; };
    auto distance = [&](float l) { return number(l, __fsub_rn(__fmul_rn(l, inverse), top)); };
    const bool once = fabsf(top) < 65536.0f;
    auto distance_once = [&](float l) { return once ? fmaf(l, inverse, -top) : distance(l); };
    const bool by_k = k > 0 && k < vocab, by_floor = floor > 0.0;
    if (!(by_k || by_floor || p < 1.0)) {
        // ---- in the order of ids: a warp has a run of tokens
        const int part = ((count + kWarps - 1) / kWarps + 31) & ~31;
        const int begin = min(count, row.warp() * part), end = min(count, begin + part);
        double mine = 0.0;
        for (int i = begin + row.lane(); i < end; i += 32) mine += weight_of(distance_once(s[i]), sh.table);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (row.lane() == 0) sh.sums[row.warp()] = mine;
        __syncthreads();
        double here = 0.0;
        for (int w = 0; w < kWarps; ++w) here += sh.sums[w];
        if (t == 0) sh.mass[0] = here;
        row.meet();
        double all = 0.0, before = 0.0;
        for (int b = 0; b < blocks; ++b) {
            const double m = blocks > 1 ? peer(&sh.mass[0], b) : here;
            if (b < block) before += m;
            all += m;
        }
        const double target = u * all;
        // the block, and in it the warp, that passes the target; should rounding leave none, the last with any weight
        int owner = -1, spare = 0;
        double run = 0.0;
        for (int b = 0; b < blocks; ++b) {
            const double m = blocks > 1 ? peer(&sh.mass[0], b) : here;
            run += m;
            if (owner < 0 && run > target) owner = b;
            if (m > 0.0) spare = b;
        }
        if (owner < 0) owner = spare;
        if (block == owner) {
            int walker = -1, last = 0;
            run = before;
            double in_front = before;
            for (int w = 0; w < kWarps; ++w) {
                const double m = sh.sums[w];
                if (walker < 0 && run + m > target) walker = w, in_front = run;
                if (m > 0.0) {
                    last = w;
                    if (walker < 0) in_front = run;
                }
                run += m;
            }
            if (walker < 0) walker = last;
            if (row.warp() == walker) {
                int token = -1, some = -1;
                for (int i0 = begin; i0 < end && token < 0; i0 += 32) {
                    const int i = i0 + row.lane();
                    const double w = i < end ? weight_of(distance_once(s[i]), sh.table) : 0.0;
                    double incl = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double other = __shfl_up_sync(0xffffffffu, incl, o);
                        if (row.lane() >= o) incl += other;
                    }
                    const unsigned passed = __ballot_sync(0xffffffffu, w > 0.0 && in_front + incl > target);
                    const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
                    if (any) some = first + i0 + 31 - __clz(any);
                    if (passed) token = first + i0 + __ffs(passed) - 1;
                    in_front += __shfl_sync(0xffffffffu, incl, 31);
                }
                if (row.lane() == 0) out[r] = token >= 0 ? token : some;
            }
        }
        row.meet();
        return;
    }
    // ---- distances, counted by bins
    {
        const float d = distance(low);
        const float reach = fminf(-d, kReach);
        row.scale = reach > 0.0f ? fminf((float)kBins / reach, 1e30f) : 0.0f;
    }
    for (int b = t; b < kBins; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    const bool whole = !by_k && !by_floor;         // top_p goes by the mass of all tokens
    double mass = 0.0;
    int far = 0;
    for (int i0 = 0; i0 < count; i0 += kThreads) {
        const int i = i0 + t;
        const float l = i < count ? s[i] : -INFINITY;
        const float d = distance(l);
        const bool any = l > -INFINITY && d > -INFINITY;
        if (i < count) s[i] = any ? d : -INFINITY;
        const int b = row.bin(d);
        // (the last bin may have most of the tokens)
        far += __popc(__ballot_sync(0xffffffffu, any && b == kBins - 1));
        if (any && b < kBins - 1) atomicAdd(&sh.hist[b], 1u);
        if (whole && any) mass += weight_of(d, sh.table);
    }
    if (row.lane() == 0 && far > 0) atomicAdd(&sh.hist[kBins - 1], (uint32_t)far);
    __syncthreads();
    Bins bins;
    if (whole) {
        mass = row.row_sum(mass);
        if (blocks == 1) row.meet();
    } else {
        row.meet();
    }
    int tokens = 0;
    for (int e = 0; e < 2; ++e) {
        bins.own[e] = 0;
        for (int b = 0; b < blocks; ++b) bins.own[e] += blocks > 1 ? (int)peer_u32(&sh.hist[2 * t + e], b) : (int)sh.hist[2 * t + e];
        tokens += bins.own[e];
    }
    {
        const int before = row.sum_before(tokens, sh.counts);
        bins.cumulative[0] = before + bins.own[0];
        bins.cumulative[1] = before + tokens;
        const double unit = row.scale > 0.0f ? 1.0 / (double)row.scale : 0.0;
        if (whole) {                               // (what a bin's tokens weigh at least)
            double least[2];
            for (int e = 0; e < 2; ++e) least[e] = 2 * t + e < kBins - 1 ? bins.own[e] * exp(-(double)(2 * t + e + 1) * unit) : 0.0;
            const double low_before = row.sum_before(least[0] + least[1], sh.sums);
            bins.least[0] = low_before + least[0];
            bins.least[1] = low_before + least[0] + least[1];
        }
    }
    const float from = by_floor ? fminf(__double2float_ru(log(floor)), 0.0f) : -INFINITY;      // d of min_p
    // ---- the last bin that a kept token may be in, and how many tokens there are up to it
    {
        int edge = kBins - 1;
        for (int e = 1; e >= 0; --e) {
            const bool enough = by_k ? bins.cumulative[e] >= k : whole && bins.least[e] * (1.0 - kSpare) >= p * mass;
            if (enough) edge = min(edge, 2 * t + e);
        }
        edge = (int)__reduce_min_sync(0xffffffffu, (unsigned)edge);
        if (t == 0) sh.edge = by_floor ? row.bin(from) : kBins - 1;
        __syncthreads();
        if (row.lane() == 0) atomicMin(&sh.edge, edge);
        __syncthreads();
        edge = sh.edge;
        if (edge >> 1 == t) sh.before = bins.cumulative[edge & 1];
        __syncthreads();
        if (sh.before <= kListed) {
            int n;
            row.gather([&](float d, int) { return d > -INFINITY && row.bin(d) <= edge; }, n);
            if (block == 0) {
                uint64_t* keys = blocks == 1 ? list : list + kListed;
                if (blocks > 1) row.pull(keys, n);
                row.sort(keys, n);
                int kept = by_k ? min(n, k) : n;
                if (by_floor) {
                    int mine = 0;
                    for (int e = t; e < kept; e += kThreads) mine += distance_of(keys[e]) >= from;
                    kept = row.block_count(mine);
                }
                Ranked ranked(row, keys, kept);
                double sum = ranked.sum_through(kept - 1);
                if (p < 1.0) {
                    const int short_by = ranked.short_of((whole ? mass : sum) * p, false, 0.0);
                    kept = min(short_by + 1, kept);
                    sum = ranked.sum_through(kept - 1);
                }
                const int place = min(ranked.short_of(sum * u, true, 0.0), kept - 1);
                if (t == 0) out[r] = (int)(uint32_t)keys[place];
            }
            row.meet();
            return;
        }
    }
    // ---- more than a list holds: cut by cut.  A bin's mass is e^(-b unit) times the sum of e^(-f unit) over its tokens' places f in it,
    // and 1 - x <= e^-x <= 1 - x + x^2 / 2: with the sum of f it is known to unit^2 / 2, 1 part in 2,048 at most.
    row.meet();                                    // (everyone has read the counts)
    for (int b = t; b < kBins; b += kThreads) sh.hist[b] = 0;
    __syncthreads();
    for (int i = t; i < count; i += kThreads) {
        const int b = row.bin(s[i]);
        if (b < kBins - 1) atomicAdd(&sh.hist[b], (uint32_t)((-s[i] * row.scale - (float)b) * 65536.0f));
    }
    row.meet();
    {
        const double unit = row.scale > 0.0f ? 1.0 / (double)row.scale : 0.0;
        double high[2], least[2];
        for (int e = 0; e < 2; ++e) {
            const int b = 2 * t + e;
            double places = 0.0;
            for (int c = 0; c < blocks; ++c) places += (double)(blocks > 1 ? peer_u32(&sh.hist[b], c) : sh.hist[b]) * (1.0 / 65536);
            const double n = bins.own[e], edge = exp(-(double)b * unit);
            least[e] = b < kBins - 1 ? edge * (n - unit * (places + n * (1.0 / 65536))) : 0.0;
            high[e] = b < kBins - 1 ? edge * (n - unit * places + 0.5 * unit * unit * n) : edge * n;
        }
        const double low_before = row.sum_before(least[0] + least[1], sh.sums);
        const double high_before = row.sum_before(high[0] + high[1], sh.sums);
        bins.least[0] = low_before + least[0];
        bins.least[1] = low_before + least[0] + least[1];
        bins.most[0] = high_before + high[0];
        bins.most[1] = high_before + high[0] + high[1];
    }
    uint64_t bound = kLast;
    double sum;
    if (by_k) bound = locate(row, bins, false, (double)k, false, bound, sum);
    if (by_floor) bound = min((unsigned long long)bound, (unsigned long long)key_of(from, 0x7fffffff));
    if (!whole) {
        mass = 0.0;
        for (int i = t; i < count; i += kThreads)
            if (s[i] > -INFINITY && key_of(s[i], first + i) <= bound) mass += weight_of(s[i], sh.table);
        mass = row.row_sum(mass);
    }
    if (p < 1.0) bound = locate(row, bins, true, mass * p, false, bound, mass);
    const uint64_t drawn = locate(row, bins, true, mass * u, true, bound, sum);
    if (block == 0 && t == 0) out[r] = (int)(uint32_t)drawn;
    row.meet();                                    // no block leaves while a peer may still read its shared memory
}

}  // namespace

TB_EXPORT int tb_choose_tokens(const float* logits, int64_t stride, const float* temperature, const double* uniform, const int* top_k,
                               const double* top_p, const double* min_p, int* out, int rows, int vocab, Rules rules,
                               cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0 || rows > 65535 || vocab > kMaxBlocks * kMaxChunk || rules.room > kMaxBiases) return TB_ERR_BAD_SIZE;
    int blocks = kMaxBlocks;
    while (blocks > 1 && vocab <= blocks / 2 * 4096) blocks >>= 1;
    const int chunk = ((vocab + blocks - 1) / blocks + 127) / 128 * 128;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks, rows, 1);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = (size_t)(blocks == 1 ? kListed : 2 * kListed) * 8 + (size_t)(chunk + 4) * 4;
    config.stream = stream;
    static bool told[64];
    int device = 0;
    if (const cudaError_t err = cudaGetDevice(&device)) return (int)err;
    if (device < 0 || device >= 64 || !told[device]) {
        if (const cudaError_t err = cudaFuncSetAttribute(choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                         2 * kListed * 8 + (kMaxChunk + 4) * 4))
            return (int)err;
        if (device >= 0 && device < 64) told[device] = true;
    }
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = blocks;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // may start under the end of the head
    attribute[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = 2;
    const cudaError_t err = cudaLaunchKernelEx(&config, choose_kernel, logits, stride, temperature, uniform, top_k, top_p, min_p, out,
                                               vocab, chunk, rules);
    return err == cudaSuccess ? tb_launch_status() : (int)err;
}
