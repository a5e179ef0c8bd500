// One token a row from 32-bit logits under the row's rules (token_rules.cuh): greedy, or drawn after top-k, min-p and top-p.
//
//   T <= 0: the lowest id of the largest logit.  Else, with z = x * (1 / T) and d = max z - z, each rounded to 32 bits (the
//   arithmetic of sample_top_p_host), weights w = e^-d in 64 bits and tokens ranked by ascending d, equal ones by id:
//     kept = the first top_k of the rank; of those w >= min_p; of those the shortest beginning with mass >= top_p * their mass
//     token = the first of the rank whose cumulative weight is above u * (mass of what is kept)
//   A row without any cut is drawn from in the order of ids with d = fma(-x, 1 / T, max z), as tb_sample does (where max z is 65,536 and
//   more, at temperatures of a thousandth and below, that would leave the largest logit itself away from 0: there d as above, unless
//   the row is marked by `as_sampled` and max z is below 2^32).
//   A row with NaN or +inf, or with nothing above -inf, has no token: -1 (`as_sampled`: the one that tb_sample gives it).  Where max z
//   leaves the 32 bits' range, the largest logits have d = 0 and the others weigh nothing.
//
// A row is shared by a thread-block cluster; each block reads its part of the vocabulary once, into shared memory, and all that follows
// runs there:
//   1. rules and mask are applied, the row's largest and smallest logit found;
//   2. the tokens are counted in 1,024 bins of d, each with its place in the bin to an eighth, and where top_p goes by it the mass of
//      all is summed.  The blocks' counts are put together, of the nearest 384 bins first, as most cuts lie in those (64 rows 58.7 us,
//      with all at once 63.2; where a flat distribution needs all, 47.8 and 45.7; both before blocks left early).  Of a bin of width h
//      whose tokens lie F eighths into it the mass is e^(-b h) (n - h F / 8) but for h / 8, so the cumulative mass is known bin by bin
//      to some 0.4 %, and with it the few bins in which each cut and the draw can lie;
//   3. the tokens of those bins are listed, what weighs in front of and between them is summed in 64 bits;
//   4. one block sorts the list, and the sums in the order of the rank give every cut and the token; the others have left by then.
// Where those bins have more tokens than a list holds (great numbers of equal logits), the distance is found by halving its interval, and
// the place among those equal to it by counting them.  No sum depends on the order of atomics: those count, or fill a list that is sorted.
//
// What bounds it: of the 4 V bytes a row, read once, a call of few rows takes a small part (one row of 128,256 logits: 0.1 us of 20).
// It is a chain of some twenty dependent phases and four cluster barriers: 3 us until the logits are there, 1.5 for the largest, 4.5 for
// weights and counts (32 tokens a thread), 4 to put the blocks' counts together, 1.7 to find the bins, 3 to list, 5 for the first
// block's sort, sums and searches.  Up to 15 rows of that vocabulary take no longer (21.7 us; one block a multiprocessor), 32 take 30
// (two), and beyond that rows queue, as a row's logits fill half of eight multiprocessors' shared memory: 64 rows 57 us, 256 rows 200,
// at 1.7 instructions a cycle and a third of all warps' time at barriers.  Greedy rows and those without a cut have fewer phases (one
// row 5.9 and 10.6 us, 64 rows 17 and 35, 256 rows 62 and 113).  Reading the logits again from L2 in place of shared memory, for
// more blocks a multiprocessor, was slower (64 rows 98 us against 83 then).
#include <mutex>

#include "sample_rows.cuh"
#include "token_rules.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBlocks = 16;
constexpr int kMaxChunk = 16384;         // tokens of a block (a bin's count and sum of eighths share 32 bits)
constexpr int kBins = 1024;
constexpr int kNear = 384;               // bins that are put together first
constexpr int kListed = 4096;
constexpr int kCells = 2 * kBins;        // of the list's sort
constexpr int kCell = 16;                // entries of a cell that one thread sorts
constexpr int kTable = 256;
constexpr int kInside = 4;
constexpr int kWindows = 3;              // where the draw, top_p's cut and top_k's cut may lie
constexpr int kIds = 18;                 // bits of an id: kMaxBlocks * kMaxChunk tokens
constexpr float kWeightless = 700.0f;    // weights of tokens beyond are taken as e^-700: nothing beside the largest, 1
constexpr float kReach = 32.0f;          // the bins cover d up to 32 at most; what is beyond is in the last
// To spare in a mass that the bins bound: the bins' width and the weights of their edges are rounded to 32 bits, 2^-24 * 32 in d.
constexpr double kSpare = 1e-5;

// The bins that the draw, top_p's cut and top_k's cut may lie in, in the order of the rank; those that meet are one.
struct Windows {
    int count, expected;                 // `expected`: their tokens
    int from[kWindows], to[kWindows];
    int draw_from, draw_to, cut_from, cut_to, cut_bin;
    int end;                             // the last bin with anything kept
    int tail[kWindows], in_front;        // tokens up to the end of each window that are in windows; in front of the last, in none
};

struct Shared {
    // first the mask's words (32 tokens each); then per bin its count << 17 | sum of eighths, and behind them the tokens up to and with
    // each bin; in the end the entries of the list a cell
    alignas(16) uint32_t cells[kCells];
    double table[kTable];                // 2^(i / 256)
    uint16_t some[kWarps][64];           // tokens of a warp that are worked on together
    double sums[kWindows + 1][32];
    int counts[kWindows + 1][32];
    int listed;
    Windows windows;
    // what the other blocks of the cluster read
    float best, low;
    int first;
    double mass[2];
    int equal;
    uint64_t place;
    // what the first block is told by each: the entries of its list; the mass of what is kept in front of each window and behind the
    // one before, and behind the last
    int listed_of[kMaxBlocks];
    double gap_of[kMaxBlocks][kWindows + 1];
    double base[kWindows + 1];
    uint8_t region[kBins];               // a bin's: kInside, or the gap between windows that it is in
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

__device__ __forceinline__ void tell(int* local, uint32_t rank, int v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(peer_address(local, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void tell(double* local, uint32_t rank, double v) {
    asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(peer_address(local, rank)), "d"(v) : "memory");
}

__device__ __forceinline__ void copy16(uint32_t to, const float* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(to), "l"(from) : "memory");
}
// (NaN if either is)
__device__ __forceinline__ float max_or_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }

// e^-d for d from -700 on in 64 bits, by a table of 2^(i / 256) and the series of what is left (P. T. P. Tang, "Table-driven
// implementation of the exponential function in IEEE floating-point arithmetic", 1989): -d = (256 m + i) ln 2 / 256 + r, |r| <= ln 2 / 512,
// e^r by its series up to r^4: what is left is below 2^-54, so that a weight is as exact as 64 bits are (up to r^3 1.4e-13 was left, and 32
// rows that keep much took 48.3 us in place of 49.8).
// Beyond kWeightless (+inf among it) it is e^-700, 10^-304.
__device__ __forceinline__ double weight_of(float d, const double* table) {
    constexpr double kSteps = -256.0 / 0.693147180559945309417232121458, kStep = 0.693147180559945309417232121458 / 256.0;
    constexpr double kRound = 6755399441055744.0;                              // 1.5 * 2^52: adding it rounds to a whole number
    const double x = (double)fminf(d, kWeightless), whole = fma(x, kSteps, kRound);
    const int n = __double2loint(whole);
    const double r = fma(whole - kRound, -kStep, -x), two = table[n & (kTable - 1)];
    const double step = __hiloint2double(__double2hiint(two) + (n >> 8 << 20), __double2loint(two));
    return fma(step * r, fma(r, fma(r, fma(r, 1.0 / 24, 1.0 / 6), 0.5), 1.0), step);
}
__device__ __noinline__ double one_weight(float d, const double* table) { return weight_of(d, table); }
// The last distance that weighs anything where tb_sample works weights out: exp, a unit off at most, may round the last one to 0.  (From
// kWeightless on in units of 32-bit numbers, 2^-14 there: 20 steps reach up to 763.)
__device__ __noinline__ float last_weight() {
    int last = __float_as_int(kWeightless);
#pragma unroll 1
    for (int step = 1 << 19; step > 0; step >>= 1)
        if (exp(-(double)__int_as_float(last + step)) > 0.0) last += step;
    return __int_as_float(last);
}

// A token's place in the rank: ascending keys.
__device__ __forceinline__ uint64_t key_of(float d, int id) { return (uint64_t)__float_as_uint(d) << kIds | (uint32_t)id; }
__device__ __forceinline__ float distance_of(uint64_t key) { return __uint_as_float((uint32_t)(key >> kIds)); }
__device__ __forceinline__ int id_of(uint64_t key) { return (int)(key & ((1u << kIds) - 1)); }

// The sum of what the block's threads in front of this one bring, and of what all bring, in a fixed order.
template <typename T>
struct Sums {
    T before, all;
};
template <typename T>
__device__ __noinline__ Sums<T> sum_before(T mine, T* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    T incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T other = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += other;
    }
    const T own = __shfl_up_sync(0xffffffffu, incl, 1);
    __syncthreads();
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    // (every warp sums the warps' sums, a lane each)
    T sum = lane < kWarps ? scratch[lane] : (T)0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
    }
    const T before = __shfl_sync(0xffffffffu, sum, max(0, warp - 1)), all = __shfl_sync(0xffffffffu, sum, 31);
    return {(warp == 0 ? (T)0 : before) + (lane == 0 ? (T)0 : own), all};
}
// A count and two masses together (one pair of barriers).
struct Three {
    int n;
    double a, b;
    __device__ __forceinline__ Three up(int o) const {
        return {__shfl_up_sync(0xffffffffu, n, o), __shfl_up_sync(0xffffffffu, a, o), __shfl_up_sync(0xffffffffu, b, o)};
    }
    __device__ __forceinline__ void add(const Three& other) {
        n += other.n;
        a += other.a;
        b += other.b;
    }
};
__device__ __forceinline__ Three three_before(const Three& mine, int* counts, double* first, double* second) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Three incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Three other = incl.up(o);
        if (lane >= o) incl.add(other);
    }
    Three own = incl.up(1);
    if (lane == 31) {
        counts[warp] = incl.n;
        first[warp] = incl.a;
        second[warp] = incl.b;
    }
    __syncthreads();
    Three sum = {0, 0.0, 0.0};
    if (lane < kWarps) sum = {counts[lane], first[lane], second[lane]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Three other = sum.up(o);
        if (lane >= o) sum.add(other);
    }
    const int from = max(0, warp - 1);
    const Three before = {__shfl_sync(0xffffffffu, sum.n, from), __shfl_sync(0xffffffffu, sum.a, from), __shfl_sync(0xffffffffu, sum.b, from)};
    if (lane == 0) own = {0, 0.0, 0.0};
    if (warp > 0) own.add(before);
    return own;
}

// Sorts n keys ascending; there is room for the next power of two.
__device__ __noinline__ void sort(uint64_t* keys, int n) {
    int size = 64;
    while (size < n) size <<= 1;
#pragma unroll 1
    for (int i = n + (int)threadIdx.x; i < size; i += kThreads) keys[i] = ~0ull;
    __syncthreads();
#pragma unroll 1
    for (int run = 2; run <= size; run <<= 1)
#pragma unroll 1
        for (int step = run >> 1; step > 0; step >>= 1) {
            // (up to 32 apart a warp's pairs lie within 64 entries of its own)
#pragma unroll 1
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

// The first place of n ascending numbers that reaches `target` (`above`: is above it); n if none does.
template <typename T>
__device__ __noinline__ int first_to(const T* of, int n, T target, bool above) {
    int low = 0, high = n;
#pragma unroll 1
    while (low < high) {
        const int middle = (low + high) >> 1;
        if (above ? of[middle] > target : of[middle] >= target) high = middle; else low = middle + 1;
    }
    return low;
}

struct Row {
    Shared& sh;
    const float* s;                      // the block's logits under the rules
    int first, count;                    // its tokens: ids first ... first + count - 1
    int block, blocks, turn;
    float inverse, top, scale;           // scale: bins a unit of d

    __device__ __forceinline__ int lane() const { return threadIdx.x & 31; }
    __device__ __forceinline__ int warp() const { return threadIdx.x >> 5; }
    __device__ __forceinline__ void meet() const {                     // all threads of the cluster
        if (blocks > 1)
            asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        else
            __syncthreads();
    }
    // The cluster's last meeting in two halves: a block has read what it needs of others' shared memory, and all have.
    __device__ __forceinline__ void done() const {
        if (blocks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    }
    __device__ __forceinline__ void leave() const {
        if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    }
    __device__ __forceinline__ float distance(float l) const { return __fsub_rn(top, __fmul_rn(l, inverse)); }
    // Where a distance lies, in eighths of a bin: what stands above 2^23 in a number that is rounded down there, so that neither a
    // conversion nor a second rounding is needed (distances beyond the bins, +inf and NaN are above all of them).
    static constexpr int kOrigin = 0x4b000000;                         // 2^23
    __device__ __forceinline__ int eighth(float d) const { return __float_as_int(__fmaf_rd(d, 8.0f * scale, 8388608.0f)); }
    static __device__ __forceinline__ int behind(int bins) { return kOrigin + 8 * bins; }              // the first behind so many bins
    __device__ __forceinline__ int bin(float d) const { return min(kBins - 1, (eighth(d) - kOrigin) >> 3); }
    // (a lane each brings its warp's, or its block's, number; two places in turn: whoever writes one again has passed a barrier behind
    // everyone's reading of it)
    __device__ __forceinline__ double across(double v) const {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    __device__ double row_sum(double v) {
        v = across(v);
        __syncthreads();
        if (lane() == 0) sh.sums[0][warp()] = v;
        __syncthreads();
        v = across(lane() < kWarps ? sh.sums[0][lane()] : 0.0);
        if (blocks == 1) return v;
        if (threadIdx.x == 0) sh.mass[turn] = v;
        meet();
        v = across(lane() < blocks ? peer(&sh.mass[turn], lane()) : 0.0);
        turn ^= 1;
        return v;
    }
    // What all threads of the cluster bring, the largest or (`most` false) all bits.
    __device__ __noinline__ uint64_t row_all(uint64_t v, bool most) {
        uint64_t* scratch = reinterpret_cast<uint64_t*>(sh.sums[0]);
        auto across = [&]() {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const uint64_t other = __shfl_xor_sync(0xffffffffu, v, o);
                v = most ? (other > v ? other : v) : v | other;
            }
        };
        across();
        __syncthreads();
        if (lane() == 0) scratch[warp()] = v;
        __syncthreads();
        v = lane() < kWarps ? scratch[lane()] : 0;
        across();
        if (blocks == 1) return v;
        if (threadIdx.x == 0) sh.place = v;
        meet();
        v = lane() < blocks ? peer_u64(&sh.place, lane()) : 0;
        across();
        meet();                                                        // (the next one may be written)
        return v;
    }
    // The token that tb_sample gives a row with NaN or +inf, or with nothing above -inf (the whole cluster calls it): NaN is never the
    // largest, and without another token 0 is.  Drawn, such a row's mass is NaN and no block passes the draw: it has the last token that
    // weighs anything in the blocks of tb_sample (`apart` tokens each, 8 at most) whose weights are all numbers, else the largest.
    __device__ __noinline__ int sampled_token(float temp, int apart) {
        uint64_t mine = 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const float l = s[i] + 0.0f;                               // (-0 and 0 are equal)
            if (!(l > -INFINITY)) continue;
            const uint32_t bits = __float_as_uint(l), order = bits >> 31 ? ~bits : bits | 0x80000000u;
            const uint64_t key = (uint64_t)order << 32 | ~(uint32_t)(first + i);
            mine = key > mine ? key : mine;
        }
        const uint64_t key = row_all(mine, true);
        const uint32_t order = (uint32_t)(key >> 32);
        const float largest = key == 0 ? -INFINITY : __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order);
        const int lowest = key == 0 ? 0 : (int)~(uint32_t)key;
        if (!(temp > 0.0f)) return lowest;
        const float by = 1.0f / temp, largest_by = largest * by;
        auto weight = [&](int i) { return exp((double)fmaf(s[i], by, -largest_by)); };
        uint64_t none = 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < count; i += kThreads)
            if (isnan(weight(i))) none |= 1ull << (first + i) / apart;
        none = row_all(none, false);
        mine = 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < count; i += kThreads)
            if (!(none >> (first + i) / apart & 1) && weight(i) > 0.0) mine = first + i + 1;
        mine = row_all(mine, true);
        return mine > 0 ? (int)mine - 1 : lowest;
    }
    // The mass, or the number, of the tokens of the rank up to `place`.
    __device__ __noinline__ double through(bool mass, uint64_t place) {
        double mine = 0.0;
#pragma unroll 1
        for (int i = threadIdx.x; i < count; i += kThreads) {
            const float d = distance(s[i]);
            if (d < INFINITY && key_of(d, first + i) <= place) mine += mass ? one_weight(d, sh.table) : 1.0;
        }
        return row_sum(mine);
    }
    // The first token of the rank up to `bound` at which the mass (or, `mass` false, the count) reaches `target` (`above`: is above it);
    // if none does (rounding, or fewer tokens than asked for), the last.  It lies in bins `from` to `to`.  The whole cluster calls it and
    // has the same answer; `sum`: the measure up to it.
    __device__ __noinline__ uint64_t halve(bool mass, double target, bool above, uint64_t bound, int from, int to, double& sum) {
        auto reach = [&](double v) { return above ? v > target : v >= target; };
        sum = through(mass, bound);
        if (!reach(sum)) {
            target = sum;
            above = false;
            from = 0;
            to = kBins - 1;
        }
        // the distance (a thousandth of a bin to spare)
        const float near = scale > 0.0f ? fmaxf(0.0f, (float)from - 1e-3f) / scale : 0.0f;
        const float far = scale == 0.0f ? 0.0f : to < kBins - 1 ? ((float)to + 1.001f) / scale : INFINITY;
        constexpr uint64_t kAll = (1u << kIds) - 1;
        uint64_t low = key_of(near, 0) >> kIds, high = min((unsigned long long)key_of(far, 0), (unsigned long long)bound) >> kIds;
#pragma unroll 1
        while (low < high) {
            const uint64_t middle = low + (high - low) / 2;
            if (reach(through(mass, min((unsigned long long)bound, (unsigned long long)(middle << kIds | kAll))))) high = middle; else low = middle + 1;
        }
        // of the tokens at that distance, by id, the fewest that reach it
        const float d = distance_of(high << kIds);
        const double in_front = high > 0 ? through(mass, (high << kIds) - 1) : 0.0, each = mass ? one_weight(d, sh.table) : 1.0;
        const int part = (count + kThreads - 1) / kThreads, begin = min(count, (int)threadIdx.x * part), end = min(count, begin + part);
        auto equal = [&](int i) { return distance(s[i]) == d && key_of(d, first + i) <= bound; };
        int mine = 0;
#pragma unroll 1
        for (int i = begin; i < end; ++i) mine += equal(i);
        const Sums<int> here = sum_before(mine, sh.counts[0]);
        if (threadIdx.x == 0) sh.equal = here.all;
        meet();
        int upto = lane() < blocks ? (blocks > 1 ? peer(&sh.equal, lane()) : here.all) : 0;          // a lane a block
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane() >= o) upto += other;
        }
        const int all = __shfl_sync(0xffffffffu, upto, 31), before = block > 0 ? __shfl_sync(0xffffffffu, upto, max(0, block - 1)) : 0;
        int least = 1, most = max(1, all);
#pragma unroll 1
        while (least < most) {
            const int middle = (least + most) >> 1;
            if (reach(in_front + (double)middle * each)) most = middle; else least = middle + 1;
        }
        sum = in_front + (double)most * each;
        const int owner = max(0, __ffs(__ballot_sync(0xffffffffu, upto >= most)) - 1);
        int left = most - before - here.before;                        // (it is the thread's left-th)
        if (block == owner && left > 0 && left <= mine) {
#pragma unroll 1
            for (int i = begin; i < end; ++i)
                if (equal(i) && --left == 0) sh.place = key_of(d, first + i);
        }
        meet();
        const uint64_t found = blocks > 1 ? peer_u64(&sh.place, owner) : sh.place;
        meet();                                                        // (the next one may be written)
        return found;
    }
};

// The same among the 1,024 numbers of the bins, by a warp.
template <typename T>
__device__ __noinline__ int first_bin(const T* of, T target, bool above) {
    const int lane = threadIdx.x & 31;
    const T last = of[32 * lane + 31];
    const unsigned part = __ballot_sync(0xffffffffu, above ? last > target : last >= target);
    if (part == 0) return kBins;
    const int begin = 32 * (__ffs(part) - 1);
    const T v = of[begin + lane];
    return begin + __ffs(__ballot_sync(0xffffffffu, above ? v > target : v >= target)) - 1;
}

// grid (blocks a row, rows); the blocks of a row are one cluster.
__global__ void __launch_bounds__(kThreads, 2)
choose_kernel(const float* __restrict__ logits, int64_t stride, const float* __restrict__ temperature, const double* __restrict__ uniform,
              const int* __restrict__ top_k, const double* __restrict__ top_p, const double* __restrict__ min_p,
              const int* __restrict__ as_sampled, int* __restrict__ out, int vocab, int chunk, int apart, Rules rules) {
    __shared__ Shared sh;
    extern __shared__ uint4 dynamic[];
    pdl_wait();                                    // the logits, and the histories, come from kernels in front
    const int r = blockIdx.y, blocks = gridDim.x, block = blockIdx.x, t = threadIdx.x;
    const int first = min(vocab, block * chunk), count = min(vocab, first + chunk) - first;
    // ---- the block's tokens into shared memory; their first lies where 16-byte copies keep their alignment
    const float* x = logits + (int64_t)r * stride + first;
    const int shift = (int)((uintptr_t)x >> 2 & 3);
    uint64_t* list = reinterpret_cast<uint64_t*>(dynamic);
    float* s = reinterpret_cast<float*>(list + kListed) + shift;
    const uint32_t s_at = (uint32_t)__cvta_generic_to_shared(s);
    {
        const int head = min(count, (4 - shift) & 3), packets = (count - head) >> 2;
#pragma unroll 2
        for (int p = t; p < packets; p += kThreads) copy16(s_at + 4 * (head + 4 * p), x + head + 4 * p);
        if (t < head) copy4(s_at + 4 * t, x + t);
        const int tail = head + 4 * packets + t;
        if (tail < count) copy4(s_at + 4 * tail, x + tail);
    }
    const int slot = rules.slots != nullptr ? rules.slots[r] : -1;
    SlotRules rule = {};
    if (slot >= 0 && slot < rules.slot_count) rule = rules.table[slot];
    const float temp = temperature[r];
    const int words = (count + 31) >> 5;           // (a block begins with a word of its own)
    const bool masked = rule.kinds & kMask;
    if (masked) {
        const uint32_t* mask = rules.masks + (int64_t)slot * rules.words + (first >> 5);
        const uint32_t hist_at = (uint32_t)__cvta_generic_to_shared(sh.cells);
#pragma unroll 1
        for (int w = t; w < words; w += kThreads) copy4(hist_at + 4 * w, mask + w);
    }
    if (t < kTable) sh.table[t] = exp2((double)t / kTable);
    Row row = {sh, s, first, count, block, blocks, 0, 0.0f, 0.0f, 0.0f};
    const int lane = row.lane(), warp = row.warp();
    // ---- penalties and biases, token by token
    if (rule.kinds & (kPenalties | kBiases)) {
        const uint32_t* seen = rules.seen + (int64_t)slot * rules.words + (first >> 5);
        const int* had = rules.counts + (int64_t)slot * rules.stride + first;
        const int biases = rule.kinds & kBiases ? min(rule.biases, rules.room) : 0;
        const int* ids = rules.bias_ids + (int64_t)slot * rules.room;
        constexpr int kMine = kMaxBiases / kThreads;
        float raw[kMine];
        auto biased = [&](int e) {                 // the token of a thread's bias, -1 for none of this block's
            const int at = t + e * kThreads, id = at < biases ? ids[at] : -1;
            return id >= first && id < first + count ? id - first : -1;
        };
        // the tokens that were had are listed, so that every thread has as many: under the logits' latency
        static_assert(kMaxChunk / 32 <= kThreads && kMaxChunk <= kListed * 4, "a word a thread, and room for all tokens of a block");
        uint16_t* some = reinterpret_cast<uint16_t*>(list);
        int listed = 0, mine = 0, times = 0;
        if (rule.kinds & kPenalties) {
            uint32_t bits = t < words ? seen[t] : 0;
            if (bits != 0 && t * 32 + 32 > count) bits &= ~0u >> (t * 32 + 32 - count);
            const Sums<int> of = sum_before(__popc(bits), sh.counts[0]);
            listed = of.all;
            int at = of.before;
#pragma unroll 1
            while (bits) {
                some[at++] = (uint16_t)(t * 32 + __ffs(bits) - 1);
                bits &= bits - 1;
            }
            __syncthreads();
            mine = t < listed ? some[t] : 0;
            times = t < listed ? had[mine] : 0;
        }
        copies_done();
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kMine; ++e) raw[e] = biased(e) >= 0 ? s[biased(e)] : 0.0f;
        __syncthreads();
        if (t < listed) s[mine] = shaped_logit(s[mine], rule, true, times, 0.0f);
#pragma unroll 1
        for (int e = t + kThreads; e < listed; e += kThreads) s[some[e]] = shaped_logit(s[some[e]], rule, true, had[some[e]], 0.0f);
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kMine; ++e) {
            const int i = biased(e);
            if (i < 0) continue;
            const bool was = rule.kinds & kPenalties && seen[i >> 5] >> (i & 31) & 1;
            s[i] = shaped_logit(raw[e], rule, was, was ? had[i] : 0, rules.biases[(int64_t)slot * rules.room + t + e * kThreads]);
        }
    }
    copies_done();
    __syncthreads();
    // ---- the mask; the row's largest and smallest logit
    const bool greedy = !(temp > 0.0f);
    float best = -INFINITY, low = INFINITY;
    int lowest = 0x7fffffff;
    {
        if (masked) {
#pragma unroll 2
            for (int i = t; i < count; i += kThreads) {
                const float v = s[i];
                if (sh.cells[i >> 5] >> (i & 31) & 1) {
                    best = max_or_nan(best, v);
                    low = fminf(low, v);
                } else {
                    s[i] = -INFINITY;
                }
            }
        } else {
#pragma unroll 4
            for (int i = t; i < count; i += kThreads) {
                const float v = s[i];
                best = max_or_nan(best, v);
                low = fminf(low, v);
            }
        }
        if (greedy) {
#pragma unroll 1
            for (int i = t; i < count && lowest == 0x7fffffff; i += kThreads)
                if (s[i] == best) lowest = first + i;
        }
        float* scratch = reinterpret_cast<float*>(sh.sums);            // best, low a warp
        auto across = [&]() {                                          // (NaN is nothing's equal: a row with one has no token anyway)
            const float mine = best;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) best = max_or_nan(best, __shfl_xor_sync(0xffffffffu, best, o));
            lowest = (int)__reduce_min_sync(0xffffffffu, (unsigned)(mine == best ? lowest : 0x7fffffff));
            low = -warp_max(-low);
        };
        across();
        if (lane == 0) {
            scratch[2 * warp] = best;
            scratch[2 * warp + 1] = low;
            sh.counts[0][warp] = lowest;
        }
        __syncthreads();
        best = lane < kWarps ? scratch[2 * lane] : -INFINITY;
        low = lane < kWarps ? scratch[2 * lane + 1] : INFINITY;
        lowest = lane < kWarps ? sh.counts[0][lane] : 0x7fffffff;
        across();
        if (blocks > 1) {
            if (t == 0) {
                sh.best = best;
                sh.low = low;
                sh.first = lowest;
            }
            row.meet();
            best = lane < blocks ? peer(&sh.best, lane) : -INFINITY;
            low = lane < blocks ? peer(&sh.low, lane) : INFINITY;
            lowest = lane < blocks ? peer(&sh.first, lane) : 0x7fffffff;
            across();
        }
    }
    if (!(best < INFINITY) || best == -INFINITY || greedy) {
        int token = best < INFINITY && best > -INFINITY ? lowest : -1;
        if (token < 0 && as_sampled != nullptr && as_sampled[r] != 0) {
            Row again = row;                       // (a copy, so that the row itself stays in registers)
            token = again.sampled_token(temp, apart);
        }
        if (block == 0 && t == 0) out[r] = token;
        row.meet();                                // no block leaves while a peer may still read its shared memory
        return;
    }
    const int k = top_k != nullptr ? top_k[r] : 0;
    const double p = top_p != nullptr ? top_p[r] : 1.0, floor = min_p != nullptr ? min_p[r] : 0.0, u = uniform[r];
    bool by_k = k > 0 && k < vocab, by_floor = floor > 0.0;
    const bool uncut = !(by_k || by_floor || p < 1.0);
    row.inverse = 1.0f / temp;
    row.top = best * row.inverse;
    bool far = !(fabsf(row.top) < 65536.0f) || row.inverse == 0.0f;
    // (a row that is to have tb_sample's token has its distances, up to where the largest one's own, half a unit of max z, is 128)
    if (far && uncut && fabsf(row.top) < 4294967296.0f && row.inverse > 0.0f && as_sampled != nullptr && as_sampled[r] != 0) far = false;
    if (far) {
        // (temperatures far from 1: the distances themselves take the logits' place, negative as those are)
        const bool finite = fabsf(row.top) < INFINITY;
        for (int i = t; i < count; i += kThreads) {
            const float l = s[i];
            s[i] = l == -INFINITY ? l : finite ? -row.distance(l) : l == best ? 0.0f : -INFINITY;
        }
        low = low == -INFINITY ? low : finite ? -row.distance(low) : low == best ? 0.0f : -INFINITY;
        row.inverse = 1.0f;
        row.top = 0.0f;
        __syncthreads();
    }
    if (uncut) {
        // ---- in the order of ids: a warp has a run of tokens
        const int part = ((count + kWarps - 1) / kWarps + 31) & ~31;
        const int begin = min(count, warp * part), end = min(count, begin + part);
        // (a draw of 0 takes the first token that weighs anything; no other gets to those beyond kWeightless)
        const float last = u > 0.0 ? kWeightless : last_weight();
        auto weight = [&](float l) {
            const float d = fmaf(-l, row.inverse, row.top);
            const double w = weight_of(d, sh.table);
            return d <= last ? w : 0.0;
        };
        double mine = 0.0;
#pragma unroll 4
        for (int i = begin + lane; i < end; i += 32) mine += weight(s[i]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) sh.sums[1][warp] = mine;
        __syncthreads();
        const double here = row.across(lane < kWarps ? sh.sums[1][lane] : 0.0);
        if (t == 0) sh.mass[0] = here;
        row.meet();
        // a lane a block: the masses up to and with it
        double upto = blocks > 1 ? (lane < blocks ? peer(&sh.mass[0], lane) : 0.0) : lane == 0 ? here : 0.0;
        const bool some = upto > 0.0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double other = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += other;
        }
        __syncwarp();
        row.done();                                // (only one block goes on: the others' places are free for another row)
        const double target = u * __shfl_sync(0xffffffffu, upto, 31);
        // the block, and in it the warp, that passes the target; should rounding leave none, the last with any weight
        const unsigned past = __ballot_sync(0xffffffffu, lane < blocks && some && upto > target), any_of = __ballot_sync(0xffffffffu, some);
        const int owner = past ? __ffs(past) - 1 : 31 - __clz(any_of);
        const double before = owner > 0 ? __shfl_sync(0xffffffffu, upto, max(0, owner - 1)) : 0.0;
        if (block == owner) {
            double run = lane < kWarps ? sh.sums[1][lane] : 0.0;
            const bool any_here = run > 0.0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double other = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += other;
            }
            const unsigned past_it = __ballot_sync(0xffffffffu, lane < kWarps && any_here && before + run > target);
            const unsigned any_warp = __ballot_sync(0xffffffffu, any_here);
            const int walker = past_it ? __ffs(past_it) - 1 : 31 - __clz(any_warp);
            double in_front = before + (walker > 0 ? __shfl_sync(0xffffffffu, run, max(0, walker - 1)) : 0.0);
            if (warp == walker) {
                int token = -1, spare = -1;
                for (int i0 = begin; i0 < end && token < 0; i0 += 32) {
                    const int i = i0 + lane;
                    const double w = i < end ? weight(s[i]) : 0.0;
                    double incl = w;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double other = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += other;
                    }
                    const unsigned passed = __ballot_sync(0xffffffffu, w > 0.0 && in_front + incl > target);
                    const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
                    if (any) spare = first + i0 + 31 - __clz(any);
                    if (passed) token = first + i0 + __ffs(passed) - 1;
                    in_front += __shfl_sync(0xffffffffu, incl, 31);
                }
                if (lane == 0) out[r] = token >= 0 ? token : spare;
            }
        }
        __syncwarp();
        row.leave();
        return;
    }
    // ---- counts by bins, and the mass of all
    {
        const float reach = fminf(row.distance(low), kReach);
        row.scale = reach > 0.0f ? fminf((float)kBins / reach, 1e30f) : 0.0f;
    }
    for (int b = t; b < kBins + 32; b += kThreads) sh.cells[b] = 0;
    __syncthreads();
    const bool whole = !by_k && !by_floor;         // top_p goes by the mass of all tokens
    const float edge = by_floor ? fmaxf(__double2float_rd(-log(floor)), 0.0f) : INFINITY;      // d of min_p
    double* least = reinterpret_cast<double*>(list);                   // (the list's place: 2 * kBins numbers)
    double* most = least + kBins;
    int* upto = reinterpret_cast<int*>(sh.cells + kBins);
    double mass = 0.0;
    {
        // (without a branch: what lies beyond the bins, which may be most, goes to a cell a lane behind them; what is ruled out, d = +inf,
        // whose place is +inf or NaN, adds 0)
        const int beyond = row.behind(kBins - 1);
        auto tally = [&](float d) {
            const int at = row.eighth(d);
            atomicAdd(&sh.cells[at < beyond ? at >> 3 & (kBins - 1) : kBins + lane], at < 0x7f800000 ? 1u << 17 | (at & 7) : 0u);
        };
        if (whole) {
            auto weigh = [&](float d) {
                tally(d);
                mass += weight_of(d, sh.table);
            };
            int i = t;
#pragma unroll 1
            for (; i + 3 * kThreads < count; i += 4 * kThreads) {
#pragma unroll
                for (int u = 0; u < 4; ++u) weigh(row.distance(s[i + u * kThreads]));
            }
#pragma unroll 1
            for (; i < count; i += kThreads) weigh(row.distance(s[i]));
        } else {
#pragma unroll 4
            for (int i = t; i < count; i += kThreads) tally(row.distance(s[i]));
        }
        __syncthreads();
        if (warp == 1) {                           // the last bin is whatever lies beyond the others
            const unsigned far = __reduce_add_sync(0xffffffffu, sh.cells[kBins + lane] >> 17);
            if (lane == 0) sh.cells[kBins - 1] = far << 17;
        }
        if (whole) mass = row.row_sum(mass);
        if (!whole || blocks == 1) row.meet();
    }
    // The blocks' counts together: of the near bins first.
#pragma unroll 1
    for (int stop = kNear;; stop = kBins) {
        // tokens, and what the mass is at least and at most, up to and with each bin
        constexpr int kEach = kBins / kThreads;
        const double unit = row.scale > 0.0f ? 1.0 / (double)row.scale : 0.0;
        int n[kEach], tokens = 0;
        double a[kEach], b[kEach], lower = 0.0, upper = 0.0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int bin = kEach * t + e;
            n[e] = 0;
            a[e] = b[e] = 0.0;
            if (bin >= stop) continue;
            int eighths = 0;
            uint32_t of[kMaxBlocks];
#pragma unroll
            for (int c = 0; c < kMaxBlocks; ++c)                       // (all under way at once)
                of[c] = c < blocks ? (blocks > 1 ? peer_u32(&sh.cells[bin], c) : sh.cells[bin]) : 0;
#pragma unroll
            for (int c = 0; c < kMaxBlocks; ++c) {
                n[e] += (int)(of[c] >> 17);
                eighths += (int)(of[c] & 0x1ffff);
            }
            // the tokens' places in the bin: between `eighths` / 8 and that and n / 8 together;  1 - x <= e^-x <= 1 - x + x^2 / 2
            const double top = one_weight((float)((double)bin * unit), sh.table), m = n[e];
            a[e] = bin < kBins - 1 ? top * (m - unit * 0.125 * (eighths + m)) : 0.0;
            b[e] = bin < kBins - 1 ? top * (m - unit * 0.125 * eighths + 0.5 * unit * unit * m) : top * m;
            tokens += n[e];
            lower += a[e];
            upper += b[e];
        }
        const Three front = three_before({tokens, lower, upper}, sh.counts[1], sh.sums[1], sh.sums[2]);
        int before = front.n;
        double under = front.a, over = front.b;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            upto[kEach * t + e] = before += n[e];
            least[kEach * t + e] = (under += a[e]) * (1.0 - kSpare);
            most[kEach * t + e] = (over += b[e]) * (1.0 + kSpare);
        }
        __syncthreads();
        // does a cut lie in what was counted?
        if (stop == kBins || (whole ? least[stop - 1] >= p * mass : (by_k && upto[stop - 1] >= k) || (by_floor && row.bin(edge) < stop))) break;
    }
    // ---- the bins that the cuts and the draw may lie in
    if (warp == 0) {
        Windows of = {};
        of.end = kBins - 1;
        if (by_floor) {
            of.end = row.bin(edge);
        }
        of.cut_bin = -1;
        if (by_k) {                                // (more than there are: no cut; behind min_p's: that cuts in front of it)
            const int bin = first_bin(upto, k, false);
            if (bin <= of.end) of.cut_bin = of.end = bin;
        }
        double lo = whole ? mass : of.end > 0 ? least[of.end - 1] : 0.0, hi = whole ? mass : most[of.end];
        of.cut_from = of.cut_to = -1;
        if (p < 1.0) {
            of.cut_from = min(first_bin(most, p * lo, false), of.end);
            of.cut_to = min(first_bin(least, p * hi, false), of.end);
            // what is kept holds p of it, and no more than the token at the cut beyond that (which weighs less than its bin's edge)
            lo = p * lo;
            hi = fmin(hi, p * hi + one_weight(of.cut_from > 0 ? (float)of.cut_from / row.scale : 0.0f, sh.table));
        }
        if (whole) of.end = of.cut_to;             // (what is behind top_p's cut is in the mass already)
        of.draw_from = min(first_bin(most, u * lo, false), of.end);
        of.draw_to = min(first_bin(least, u * hi, true), of.end);
        if (lane == 0) {
            const int a[kWindows] = {of.draw_from, of.cut_from, of.cut_bin}, b[kWindows] = {of.draw_to, of.cut_to, of.cut_bin};
#pragma unroll
            for (int v = 0; v < kWindows; ++v) {
                if (a[v] < 0) continue;
                const int n = of.count;
                if (n > 0 && a[v] <= sh.windows.to[n - 1] + 1) {
                    sh.windows.from[n - 1] = min(sh.windows.from[n - 1], a[v]);
                    sh.windows.to[n - 1] = max(sh.windows.to[n - 1], b[v]);
                } else {
                    sh.windows.from[n] = a[v];
                    sh.windows.to[n] = b[v];
                    of.count = n + 1;
                }
            }
#pragma unroll 1
            for (int v = 0; v < of.count; ++v) {
                const int ahead = sh.windows.from[v] > 0 ? upto[sh.windows.from[v] - 1] : 0;
                sh.windows.in_front = ahead - of.expected;
                of.expected += upto[sh.windows.to[v]] - ahead;
                sh.windows.tail[v] = of.expected;
            }
            sh.windows.count = of.count;
            sh.windows.expected = of.expected;
            sh.windows.draw_from = of.draw_from;
            sh.windows.draw_to = of.draw_to;
            sh.windows.cut_from = of.cut_from;
            sh.windows.cut_to = of.cut_to;
            sh.windows.cut_bin = of.cut_bin;
            sh.windows.end = of.end;
            sh.listed = 0;
        }
    }
    __syncthreads();                               // (from here on the list's place is free)
    const int windows = sh.windows.count, end = sh.windows.end, upto_end = upto[end];
    by_k = sh.windows.cut_bin >= 0;
    int from[kWindows], to[kWindows];
#pragma unroll
    for (int v = 0; v < kWindows; ++v) {
        from[v] = v < windows ? sh.windows.from[v] : kBins;
        to[v] = v < windows ? sh.windows.to[v] : kBins;
    }
    if (sh.windows.expected <= kListed) {
        // ---- list the windows' tokens, sum what lies in front of and between them
#pragma unroll
        for (int e = 0; e < kBins / kThreads; ++e) {
            const int bin = t + e * kThreads;
            int region = windows;
#pragma unroll
            for (int v = kWindows - 1; v >= 0; --v) region = bin < from[v] ? min(region, v) : bin <= to[v] ? kInside : region;
            sh.region[bin] = (uint8_t)region;
        }
        __syncthreads();
        double gap[kWindows + 1] = {0.0, 0.0, 0.0, 0.0};
        auto take = [&](int i, float d) {
            const int region = sh.region[row.bin(d)];
            if (region == kInside) {
                list[atomicAdd(&sh.listed, 1)] = key_of(d, first + i);                       // (any order: it is sorted)
            } else {
                const double weight = weight_of(d, sh.table);
                if (region == 0) gap[0] += weight;
                if (region == 1) gap[1] += weight;
                if (region == 2) gap[2] += weight;
                if (region == 3) gap[3] += weight;
            }
        };
        const int stop = end < kBins - 1 ? row.behind(end + 1) : 0x7fffffff;
        const float limit = fminf(edge, 3.402823466e38f);
        if (upto_end > vocab / 4) {
#pragma unroll 2
            for (int i = t; i < count; i += kThreads) {
                const float d = row.distance(s[i]);
                if (row.eighth(d) < stop && d <= limit) take(i, d);
            }
        } else {
            uint32_t mine = 0;                     // a bit a token of the thread's that is kept, or may be
#pragma unroll 4
            for (int i = t, e = 0; i < count; i += kThreads, ++e) {
                const float d = row.distance(s[i]);
                mine |= row.eighth(d) < stop && d <= limit ? 1u << e : 0u;
            }
            // few of a warp's are, and some lanes have more than others: they are worked on side by side, up to 64 together
            uint16_t* some = sh.some[warp];
            int place = __popc(mine);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, place, o);
                if (lane >= o) place += other;
            }
            const int total = __shfl_sync(0xffffffffu, place, 31);
            place -= __popc(mine);
#pragma unroll 1
            for (int base = 0; base < total; base += 64) {
#pragma unroll 1
                while (mine && place < base + 64) {
                    some[place++ - base] = (uint16_t)(t + (__ffs(mine) - 1) * kThreads);
                    mine &= mine - 1;
                }
                __syncwarp();
#pragma unroll 1
                for (int e = lane; e < min(64, total - base); e += 32) take(some[e], row.distance(s[some[e]]));
                __syncwarp();
            }
        }
        __syncwarp();
        // four sums over a warp at once: each exchange with a lane half as far away leaves half as many to a lane
        {
            const bool upper = lane & 16, odd = lane & 8;
            const double a = upper ? gap[2] : gap[0], b = upper ? gap[3] : gap[1];
            const double c = a + __shfl_xor_sync(0xffffffffu, upper ? gap[0] : gap[2], 16);
            const double d = b + __shfl_xor_sync(0xffffffffu, upper ? gap[1] : gap[3], 16);
            double sum = (odd ? d : c) + __shfl_xor_sync(0xffffffffu, odd ? c : d, 8);
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if ((lane & 7) == 0) sh.sums[(upper ? 2 : 0) + (odd ? 1 : 0)][warp] = sum;
        }
        __syncthreads();
        // (each block tells the first; what another one reads in its turn stays where it is until the end)
        if (t <= windows) {
            double sum = 0.0;
#pragma unroll 8
            for (int w = 0; w < kWarps; ++w) sum += sh.sums[t][w];
            tell(&sh.gap_of[block][t], 0, sum);
        } else if (t == 64) {
            tell(&sh.listed_of[block], 0, sh.listed);
        }
        row.meet();
        if (block == 0) {
            // ---- the whole row's list, over the place of the block's logits, and behind it room for it in order
            uint64_t* keys = reinterpret_cast<uint64_t*>(s - shift);
            uint64_t* sorted = keys + kListed;
            if (t == 0) {
                double base = 0.0;
#pragma unroll 1
                for (int v = 0; v <= windows; ++v) {
#pragma unroll 4
                    for (int b = 0; b < blocks; ++b) base += sh.gap_of[b][v];
                    sh.base[v] = base;
                }
            }
            int before = lane < blocks ? sh.listed_of[lane] : 0;       // a lane a block: the entries up to and with it
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int other = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += other;
            }
            const int n = __shfl_sync(0xffffffffu, before, 31);
#pragma unroll 1
            for (int e0 = 0; e0 < n; e0 += kThreads) {
                const int e = e0 + t;
                int b = 0, begin = 0;
#pragma unroll
                for (int c = 0; c < kMaxBlocks - 1; ++c) {
                    const int past = __shfl_sync(0xffffffffu, before, c);
                    if (e >= past) {
                        b = c + 1;
                        begin = past;
                    }
                }
                if (e < n) keys[e] = blocks > 1 ? peer_u64(list + e - begin, b) : list[e];
            }
            __syncwarp();
            // (the other blocks leave while this one sorts, their places are the next rows': 256 rows 200 us, 216 with all until the end)
            row.done();
            // ---- sorted by cells: a bin of a window is so many of them that there are some 2,048
            int bins = 0, offset[kWindows];
#pragma unroll
            for (int v = 0; v < kWindows; ++v) {
                offset[v] = bins - from[v];
                bins += v < windows ? to[v] - from[v] + 1 : 0;
            }
            const int fine = kCells / bins;
            auto cell_of = [&](uint64_t key) {
                const float d = distance_of(key), at = d * row.scale;
                const int bin = row.bin(d);
                const int v = (bin > to[0] ? 1 : 0) + (bin > to[1] ? 1 : 0);
                return (bin + (v == 0 ? offset[0] : v == 1 ? offset[1] : offset[2])) * fine +
                       max(0, min(fine - 1, (int)((at - (float)bin) * (float)fine)));
            };
            constexpr int kEach = kCells / kThreads;
            int* cells = reinterpret_cast<int*>(sh.cells);
#pragma unroll
            for (int e = 0; e < kEach; ++e) cells[kEach * t + e] = 0;
            __syncthreads();
#pragma unroll 1
            for (int e = t; e < n; e += kThreads) atomicAdd(&cells[cell_of(keys[e])], 1);
            __syncthreads();
            int mine[kEach], own = 0, most_of = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                mine[e] = cells[kEach * t + e];
                own += mine[e];
                most_of = max(most_of, mine[e]);
            }
            const int begin = sum_before(own, sh.counts[0]).before;
            int at = begin;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                cells[kEach * t + e] = at;
                at += mine[e];
            }
            const bool crowded = __syncthreads_or(most_of > kCell);
#pragma unroll 1
            for (int e = t; e < n; e += kThreads) sorted[atomicAdd(&cells[cell_of(keys[e])], 1)] = keys[e];
            __syncthreads();
            if (crowded) {
                sort(sorted, n);
            } else {
                at = begin;
#pragma unroll 1
                for (int e = 0; e < kEach; ++e) {
#pragma unroll 1
                    for (int i = 1; i < mine[e]; ++i) {
                        const uint64_t key = sorted[at + i];
                        int j = at + i;
#pragma unroll 1
                        for (; j > at && sorted[j - 1] > key; --j) sorted[j] = sorted[j - 1];
                        sorted[j] = key;
                    }
                    at += mine[e];
                }
                __syncthreads();
            }
            // ---- sums in the order of the rank, and with them the cuts and the token
            double* sums = reinterpret_cast<double*>(keys);
            const int each = (n + kThreads - 1) / kThreads, first_of = min(n, t * each), last_of = min(n, first_of + each);
            double weight = 0.0;
#pragma unroll 1
            for (int e = first_of; e < last_of; ++e) {
                const double w = one_weight(distance_of(sorted[e]), sh.table);
                sums[e] = w;
                weight += w;
            }
            const Sums<double> of = sum_before(weight, sh.sums[0]);
            double run = of.before;
#pragma unroll 1
            for (int e = first_of; e < last_of; ++e) {
                run += sums[e];
                const int v = (e >= sh.windows.tail[0] ? 1 : 0) + (windows > 1 && e >= sh.windows.tail[1] ? 1 : 0);
                sums[e] = sh.base[min(v, windows - 1)] + run;
            }
            __syncthreads();
            // A launch behind is let in only now (by the other blocks' leaving, and here): one that may place its rows while most blocks
            // have left and the first ones not, finds worse places for them (32 rows of top-p in launches like this 35.6 us, 29.6 so).
            pdl_trigger();
            if (t == 0) {
                int kept = n;
                double total = of.all + sh.base[windows];
                if (by_k && k - sh.windows.in_front < n) {
                    kept = max(1, k - sh.windows.in_front);
                    total = sums[kept - 1];
                }
                if (whole) total = mass;
                if (p < 1.0) {
                    kept = min(first_to(sums, kept, p * total, false) + 1, kept);
                    total = sums[kept - 1];
                }
                out[r] = id_of(sorted[max(0, min(first_to(sums, kept, u * total, true), kept - 1))]);
            }
        } else {
            row.done();
        }
        __syncwarp();
        row.leave();
        return;
    } else {
        // ---- more than a list holds: cut by cut  (on a copy, so that the row itself stays in registers)
        Row again = row;
        again.meet();                              // (the places of the sums are free)
        uint64_t bound = key_of(INFINITY, (1 << kIds) - 1);
        double sum;
        if (by_k) bound = again.halve(false, (double)k, false, bound, end, end, sum);
        if (by_floor) bound = min((unsigned long long)bound, (unsigned long long)key_of(edge, (1 << kIds) - 1));
        if (!whole) mass = again.through(true, bound);
        if (p < 1.0) {
            bound = again.halve(true, mass * p, false, bound, sh.windows.cut_from, sh.windows.cut_to, sum);
            mass = sum;
        }
        const uint64_t picked = again.halve(true, mass * u, true, bound, sh.windows.draw_from, sh.windows.draw_to, sum);
        if (block == 0 && t == 0) out[r] = id_of(picked);
    }
    row.meet();                                    // no block leaves while a peer may still read its shared memory
}

int launch_rows(int rows, int vocab, int blocks, cudaStream_t stream, const float* logits, int64_t stride, const float* temperature,
                const double* uniform, const int* top_k, const double* top_p, const double* min_p, const int* as_sampled, int* out,
                const Rules& rules) {
    const int chunk = ((vocab + blocks - 1) / blocks + 127) / 128 * 128;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = blocks;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // may start under the end of the head
    attribute[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks, rows, 1);
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    config.attrs = attribute;
    config.numAttrs = 2;
    // the list; behind it the logits, in whose place the first block later has the row's list and its sums
    const size_t logits_at = kListed * 8, space = (size_t)(chunk + 4) * 4, later = 2 * kListed * 8;
    // Once a device: what the kernel may have, and how many rows of so many blocks find a multiprocessor a block at the same time.  Those
    // are kept apart, by shared memory that they do not use (12 rows of 128,256 logits 22.6 us, 28.8 with two blocks a multiprocessor).
    constexpr size_t kAlone = 120 * 1024;
    static std::mutex lock;
    static int rows_apart[64][kMaxBlocks + 1];
    int device = 0, apart = 0;
    if (const cudaError_t err = cudaGetDevice(&device)) return (int)err;
    if (device < 0 || device >= 64) return TB_ERR_BAD_SIZE;
    {
        std::lock_guard<std::mutex> guard(lock);
        if (rows_apart[device][blocks] == 0) {
            if (const cudaError_t err = cudaFuncSetAttribute(choose_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kAlone))
                return (int)err;
            if (const cudaError_t err = cudaFuncSetAttribute(choose_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1))
                return (int)err;
            config.dynamicSmemBytes = kAlone;
            int clusters = 0;
            if (const cudaError_t err = cudaOccupancyMaxActiveClusters(&clusters, choose_kernel, &config)) return (int)err;
            rows_apart[device][blocks] = 1 + clusters;                 // (0: not asked yet)
        }
        apart = rows_apart[device][blocks] - 1;
    }
    config.dynamicSmemBytes = logits_at + (space > later ? space : later);
    if (blocks > 1 && rows <= apart) config.dynamicSmemBytes = kAlone;
    const cudaError_t err = cudaLaunchKernelEx(&config, choose_kernel, logits, stride, temperature, uniform, top_k, top_p, min_p,
                                               as_sampled, out, vocab, chunk, sample_chunk(sample_blocks(rows, vocab), vocab), rules);
    return err == cudaSuccess ? tb_launch_status() : (int)err;
}

int sm_count() {
    static int sms = 0;
    if (sms == 0) {
        int device = 0;
        cudaGetDevice(&device);
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 1;
    }
    return sms;
}

}  // namespace

TB_EXPORT int tb_choose_tokens(const float* logits, int64_t stride, const float* temperature, const double* uniform, const int* top_k,
                               const double* top_p, const double* min_p, const int* as_sampled, int* out, int rows, int vocab,
                               Rules rules, cudaStream_t stream) {
    if (rows == 0) return 0;
    if (vocab <= 0 || rows < 0 || rows > 65535 || vocab > kMaxBlocks * kMaxChunk || rules.room > kMaxBiases) return TB_ERR_BAD_SIZE;
    // As few blocks a row as hold it, and up to eight while each has a multiprocessor of its own and 2,048 tokens.  (Device time, 8 / 4
    // blocks a row: 8 rows of 50,257 logits 20.7 / 22.5 us, 64 rows 56 / 31; 16 blocks of 128,256 logits: 1 row 27.6 us, 28.7 with 8, 8
    // rows 39, 30 with 8, as few clusters of 16 fit the chip.  Blocks of 1,024 threads: 16 rows 56 us, 40 with 512, two blocks a
    // multiprocessor.)
    int blocks = (vocab + kMaxChunk - 1) / kMaxChunk;
    const int more = min(min(8, sm_count() / rows), vocab / 2048);
    if (blocks < more) blocks = more;
    return launch_rows(rows, vocab, blocks, stream, logits, stride, temperature, uniform, top_k, top_p, min_p, as_sampled, out, rules);
}
