// Log probabilities of given tokens, the entropy and the most probable alternatives, from 32-bit logits in one pass.
//
// For a row x of V logits, a token t and k alternatives:
//   m = max x,  S = sum e^(x_i - m),  T = sum (x_i - m) e^(x_i - m)
//   logprob = x_t - m - ln S        entropy = ln S - T / S        alternative j: its id, and x_id - m - ln S
// Alternatives go by descending logit, equal ones by ascending id.  A logit of -inf has probability 0 (log probability
// -inf) and adds nothing to S, T and the entropy; a NaN or +inf in a row makes its numbers NaN.  A token outside the
// vocabulary has log probability NaN.
//
// Bound by HBM: 4 V bytes a row, read once.  A row is shared by a thread-block cluster of 1 to 8 blocks (a contiguous
// part each); a block takes its part in chunks of sixteen logits a thread, two chunks' asynchronous copies under way while one is
// worked on in registers.  Many rows: blocks of 256 threads, four a multiprocessor, so that one row's beginning and end run under the
// others' loads (1,536 rows of 128,256 logits, one alternative: 133 us, 0.92 of the measured copy rate; 143 where the clocks have fallen
// under minutes of load); few rows: blocks of 1,024, up to eight a row (64 rows of that vocabulary, 20 alternatives, two blocks of four
// chunks a row: 14.1 us, of which the 33 MB are 5.1, the rest the start, the bound, the second reading and the exchange of a
// cluster).  Of a chunk
//   * every thread adds its numbers to a maximum, S and T of its own (rescaled when its maximum rises), all in 32 bits;
//     they meet once, at the end, in a fixed order, so a row's numbers do not depend on the timing;
//   * every eight threads leave the largest of their 128 logits.  No block waits for anything inside the loop.
// The alternatives come behind it: the k-th largest (or so) of those maxima is a bound that at least k logits reach, the few groups
// of 128 that reach it are read once more (from L2), and what reaches it is ranked (an entry's rank is the number of entries in front
// of it).  Where more logits reach the bound than the list holds (logits in order, a vocabulary of few groups, masks), the
// interval of their bit patterns is halved, reading those groups each time, until few enough do; and if equal numbers leave no
// such bound, what lies above is taken and of the equal ones those of lowest id.
#include "common.cuh"

namespace {

constexpr int kPackets = 4;                        // 16-byte loads of a thread and chunk
constexpr int kEach = 4 * kPackets;                // logits of a thread and chunk
constexpr int kMaxTop = 64;
constexpr int kListed = 512;                       // entries of the list
constexpr int kGroup = 8;                          // threads whose largest logit is kept
constexpr int kMaxGroups = 2048;                   // of a block (a longer part: of so many chunks together that they fit)
constexpr int kSlots = 2;                          // chunks under way
constexpr int kMaxBlocks = 8;
constexpr int kNobody = 0x7fffffff;                // the id of an entry that is none
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1024.0f;                   // e^x is 0 in 32 bits from here on down

struct Shared {
    float value[kListed];
    int id[kListed];
    float best_value[kMaxTop];                     // k entries in order, behind those there are (-inf, kNobody)
    int best_id[kMaxTop];
    alignas(16) uint32_t group[kMaxGroups];        // the groups' largest logits, as `ordered` has them
    int16_t reaching[kMaxGroups];                  // the groups that reach the bound
    float warp_stat[32][3];
    int warp_count[32];
    uint32_t bound;
    float stat[3];                                 // this block's m, S, T
    int count, groups;                             // entries of the list, of `reaching`
};

// floats as unsigned numbers of the same order (-inf smallest; NaN never gets here)
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ float exp2_of(float x) {       // 2^x, relative error about 2^-22, 0 below 2^-126
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Blackwell's packed 32-bit pairs: one instruction for two numbers.  With a scalar loop the kernel was bound by its instructions where
// the clocks fall under load (1,536 rows: 142 to 145 us then, 132 in the first seconds).
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// (m, S, T) of a warp's lanes together, in every lane; a lane with nothing brings (-inf, 0, 0).  Every lane is brought to the common
// maximum once and then S and T are summed.
__device__ __forceinline__ void meet(float& m, float& s, float& t) {
    const float top = from_ordered(__reduce_max_sync(0xffffffffu, ordered(m)));
    if (top > -INFINITY) {                         // (nothing anywhere: S and T are 0, or NaN, as they are)
        // (where e^(m - top) is 0, the distance must not make an infinity of what it is multiplied by; an infinite top gives NaN)
        const float d = m - top, a = exp2_of(d * kLog2e);
        t = (t + s * fmaxf(d, kFar)) * a;
        s *= a;
    }
    m = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
    }
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ uint32_t peer_u32(const void* local, uint32_t rank) {
    uint32_t remote, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n"
                 : "=r"(remote) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(remote) : "memory");
    return v;
}

// The k best of the list's n entries, in order, into best_value / best_id: the rank of an entry is the number of entries in front of
// it.  Every thread calls this; the list is whole (a barrier in front).
// (Not inlined: the second call finds its instructions there.)
template <int THREADS>
__device__ __noinline__ void cut(Shared& sh, int n, int k) {
    int shift = 3;                                 // 2^shift threads count for one entry
    while (shift > 0 && (n << shift) > THREADS) --shift;
    const int share = 1 << shift;
    if ((int)threadIdx.x >= n && (int)threadIdx.x < k) {
        sh.best_value[threadIdx.x] = -INFINITY;
        sh.best_id[threadIdx.x] = kNobody;
    }
    const int warp_first = threadIdx.x & ~31;      // (a warp without an entry has nothing to do)
    for (int base = 0; base + (warp_first >> shift) < n; base += THREADS >> shift) {
        const int e = base + ((int)threadIdx.x >> shift), part = (int)threadIdx.x & (share - 1);
        const bool mine = e < n;
        const float v = mine ? sh.value[e] : 0.0f;
        const int id = mine ? sh.id[e] : 0;
        int rank = 0;
        if (mine) {
#pragma unroll 4
            for (int j = part; j < n; j += share) {
                const float o = sh.value[j];
                rank += o > v || (o == v && sh.id[j] < id) ? 1 : 0;
            }
        }
        for (int o = share / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
        if (mine && part == 0 && rank < k) {
            sh.best_value[rank] = v;
            sh.best_id[rank] = id;
        }
    }
    __syncthreads();
}

template <int THREADS>
__device__ __forceinline__ int sum_before(Shared& sh, int mine, int& all) {      // exclusive sum over the block's threads
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += other;
    }
    __syncthreads();
    if (lane == 31) sh.warp_count[warp] = incl;
    __syncthreads();
    int before = incl - mine;
    all = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += sh.warp_count[w];
        all += sh.warp_count[w];
    }
    return before;
}

// Puts what may be among the k best of the block's logits into the list and returns how many that are (at least k, or all above
// -inf if they are fewer; at most kListed).  The groups' largest logits, the block's m and zeroed counts are there.
template <int THREADS>
__device__ int find_best(Shared& sh, const float* base, int ahead, int end, int first, int chunks, int span, int groups,
                         int k) {
    constexpr int kChunk = kEach * THREADS, kGroups = THREADS / kGroup;
    // low: what at least k logits reach, or all above -inf; high: what fewer than k groups (later: logits) reach
    const uint32_t nothing = ordered(-INFINITY) + 1;
    if (threadIdx.x < 32) {
        // one warp looks for the bound (a barrier a round cost the block four times as much): it begins at the smallest of its lanes'
        // largest, or for k above 32 second largest, groups, which 32, or 64, groups reach
        const int lane = threadIdx.x;
        // (four at a time: what is behind the last is 0 up to a multiple of 128)
        const uint4* four = reinterpret_cast<const uint4*>(sh.group);
        uint32_t one = 0, two = 0;
        auto meet_one = [&](uint32_t v) {
            two = max(two, min(one, v));
            one = max(one, v);
        };
#pragma unroll 4
        for (int g = lane; g * 4 < groups; g += 32) {
            const uint4 v = four[g];
            meet_one(v.x);
            meet_one(v.y);
            meet_one(v.z);
            meet_one(v.w);
        }
        uint32_t low = max(nothing, __reduce_min_sync(0xffffffffu, k <= 32 ? one : two));
        uint32_t high = __reduce_max_sync(0xffffffffu, one) + 1;
        while (high > low + 1) {
            const uint32_t middle = low + (high - low) / 2;
            int reach = 0;
#pragma unroll 8
            for (int g = lane; g * 4 < groups; g += 32) {
                const uint4 v = four[g];
                reach += (v.x >= middle ? 1 : 0) + (v.y >= middle ? 1 : 0) + (v.z >= middle ? 1 : 0) + (v.w >= middle ? 1 : 0);
            }
            reach = __reduce_add_sync(0xffffffffu, reach);
            if (reach < k) {
                high = middle;
            } else {
                low = middle;
                if (reach <= k + k / 4) break;
            }
        }
        if (lane == 0) sh.bound = low;
    }
    __syncthreads();
    uint32_t low = sh.bound, high;
    for (int g = threadIdx.x; g < groups; g += THREADS)
        if (sh.group[g] >= low) sh.reaching[atomicAdd(&sh.groups, 1)] = (int16_t)g;
    __syncthreads();
    const int reaching = sh.groups;
    // every logit of the groups that reach `low`, a group of threads each: take(logit, id)
    auto walk = [&](auto take) {
        for (int e = threadIdx.x / kGroup; e < reaching; e += kGroups) {
            const int g = sh.reaching[e], c0 = g / kGroups * span, thread = g % kGroups * kGroup + (int)threadIdx.x % kGroup;
            for (int c = c0; c < min(chunks, c0 + span); ++c) {
                float x[kEach];
#pragma unroll
                for (int u = 0; u < kPackets; ++u) {
                    const int i = c * kChunk + (u * THREADS + thread) * 4;
                    if (i >= ahead && i + 4 <= end) {
                        *reinterpret_cast<float4*>(x + 4 * u) = *reinterpret_cast<const float4*>(base + i);
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[4 * u + j] = i + j >= ahead && i + j < end ? base[i + j] : -INFINITY;
                    }
                }
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    take(x[i], first + c * kChunk + ((i >> 2) * THREADS + thread) * 4 + (i & 3) - ahead);
            }
        }
    };
    auto add = [&](float x, int id) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kListed) {
            sh.value[at] = x;
            sh.id[at] = id;
        }
    };
    float cutoff = from_ordered(low);
    walk([&](float x, int id) { if (x >= cutoff) add(x, id); });
    __syncthreads();
    int n = sh.count;
    if (n <= kListed) return n;
    // more than the list holds
    high = ordered(sh.stat[0] + 0.0f) + 1;
    while (high > low + 1) {
        const uint32_t middle = low + (high - low) / 2;
        const float at_least = from_ordered(middle);
        __syncthreads();                           // (everyone has read the count)
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        int mine = 0;
        walk([&](float x, int) { mine += x >= at_least ? 1 : 0; });
        __syncwarp();
        mine = __reduce_add_sync(0xffffffffu, mine);
        if ((threadIdx.x & 31) == 0) atomicAdd(&sh.count, mine);
        __syncthreads();
        n = sh.count;
        if (n < k) {
            high = middle;
        } else {
            low = middle;
            if (n <= kListed) break;
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    cutoff = from_ordered(low);
    if (high > low + 1) {
        walk([&](float x, int id) { if (x >= cutoff) add(x, id); });
        __syncthreads();
        return sh.count;
    }
    // fewer than k logits are larger than `cutoff`, more than fit equal to it: the larger ones, and of the equal ones the first k by
    // id (packets of a lower u come first, then lower threads)
    walk([&](float x, int id) { if (x > cutoff) add(x, id); });
    int taken = 0;
    for (int c = 0; c < chunks && taken < k; ++c) {
        for (int u = 0; u < kPackets && taken < k; ++u) {
            const int i = c * kChunk + (u * THREADS + (int)threadIdx.x) * 4;
            float x[4];
            int equal = 0, all;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[j] = i + j >= ahead && i + j < end ? base[i + j] : -INFINITY;
                equal += x[j] == cutoff ? 1 : 0;
            }
            int at = taken + sum_before<THREADS>(sh, equal, all);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (x[j] != cutoff) continue;
                if (at < k) add(x[j], first + i + j - ahead);
                ++at;
            }
            taken += all;
        }
    }
    __syncthreads();
    return sh.count;
}

// grid: rows * blocks; the blocks of a row are one cluster.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logprobs_kernel(const float* __restrict__ logits, int64_t stride, const int* __restrict__ tokens,
                float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_value,
                int* __restrict__ top_id, int vocab, int k, int blocks, int part) {
    constexpr int WARPS = THREADS / 32, kChunk = kEach * THREADS, kGroups = THREADS / kGroup;
    extern __shared__ float4 ring[];               // [kSlots][kPackets][THREADS]
    __shared__ Shared sh;
    pdl_trigger();
    const int64_t r = blockIdx.x / blocks;
    const int block = blockIdx.x % blocks;
    const float* row = logits + r * stride;
    // the block's part, [first, last), as 16-byte packets of the row from the boundary at or in front of its first logit on
    const int first = min(vocab, block * part), last = min(vocab, first + part);
    const int ahead = (int)(((uintptr_t)(row + first) >> 2) & 3);
    const float* base = row + first - ahead;       // (only packets that lie wholly inside the part are read as such)
    const int end = last - first + ahead;          // logits are base[ahead .. end)
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();                                    // the logits come from the kernel in front
    // A chunk's packets on their way into this thread's own places of ring slot c % kSlots (nobody else reads them: no barrier).  A slot
    // is free as soon as its chunk is in registers, so kSlots chunks are under way while one is worked on.
    auto fetch = [&](int c) {
#pragma unroll
        for (int u = 0; u < kPackets; ++u) {
            const int i = c * kChunk + (u * THREADS + (int)threadIdx.x) * 4;
            float4* to = ring + (c % kSlots * kPackets + u) * THREADS + threadIdx.x;
            if (i >= ahead && i + 4 <= end) {
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                             ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(base + i) : "memory");
            } else {
                to->x = i >= ahead && i < end ? base[i] : -INFINITY;
                to->y = i + 1 >= ahead && i + 1 < end ? base[i + 1] : -INFINITY;
                to->z = i + 2 >= ahead && i + 2 < end ? base[i + 2] : -INFINITY;
                to->w = i + 3 >= ahead && i + 3 < end ? base[i + 3] : -INFINITY;
            }
        }
    };

    float m = -INFINITY, s = 0.0f, t = 0.0f;
    const int chunks = (end + kChunk - 1) / kChunk;
    const int span = max(1, (chunks * kGroups + kMaxGroups - 1) / kMaxGroups);       // chunks that a group's largest is taken over (1 up to 262,144 logits of a part)
    const int group = threadIdx.x / kGroup;
    const int groups = (chunks + span - 1) / span * kGroups;
    if ((int)threadIdx.x < ((groups + 127) & ~127) - groups) sh.group[groups + threadIdx.x] = 0;
    float largest = -INFINITY;
    const int token = block == 0 && threadIdx.x == 0 ? tokens[r] : -1;
#pragma unroll
    for (int c = 0; c < kSlots; ++c) {
        if (c < chunks) fetch(c);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const float given = token >= 0 && token < vocab ? row[token] : NAN;
    for (int c = 0; c < chunks; ++c) {
        float x[kEach];
        asm volatile("cp.async.wait_group %0;" ::"n"(kSlots - 1) : "memory");
#pragma unroll
        for (int u = 0; u < kPackets; ++u)
            *reinterpret_cast<float4*>(x + 4 * u) = ring[(c % kSlots * kPackets + u) * THREADS + threadIdx.x];
        if (c + kSlots < chunks) fetch(c + kSlots);
        asm volatile("cp.async.commit_group;" ::: "memory");
        float top = max3(x[0], x[1], x[2]);
#pragma unroll
        for (int i = 3; i + 1 < kEach; i += 2) top = max3(top, x[i], x[i + 1]);
        top = fmaxf(top, x[kEach - 1]);
        top = top > -INFINITY ? top + 0.0f : -INFINITY;   // (sixteen NaNs; -0 is +0, as comparisons have it)
        if (top > m) {
            if (m > -INFINITY) {
                const float d = m - top, a = exp2_of(d * kLog2e);
                t = (t + s * fmaxf(d, kFar)) * a;
                s *= a;
            }
            m = top;
        }
        const float low = m > -INFINITY ? m : 0.0f;
        const uint64_t minus_low = pack2(-low, -low), log2e = pack2(kLog2e, kLog2e);
        uint64_t s2 = 0, t2 = 0;                   // (two zeros each)
#pragma unroll
        for (int i = 0; i < kEach; i += 2) {
            const uint64_t d = add2(pack2(x[i], x[i + 1]), minus_low);
            float y0, y1, d0, d1;
            unpack2(mul2(d, log2e), y0, y1);
            unpack2(d, d0, d1);
            const uint64_t e = pack2(exp2_of(y0), exp2_of(y1));
            s2 = add2(s2, e);
            t2 = fma2(pack2(fmaxf(d0, kFar), fmaxf(d1, kFar)), e, t2);       // (-inf adds nothing, a NaN comes in by e)
        }
        float s0, s1, t0, t1;
        unpack2(s2, s0, s1);
        unpack2(t2, t0, t1);
        s += s0 + s1;
        t += t0 + t1;
        if (k == 0) continue;
        largest = fmaxf(largest, top);
        if ((c + 1) % span == 0 || c + 1 == chunks) {
#pragma unroll
            for (int o = 1; o < kGroup; o <<= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
            if (threadIdx.x % kGroup == 0) sh.group[c / span * kGroups + group] = ordered(largest);
            largest = -INFINITY;
        }
    }

    // the block's sums, in an order of lanes and warps that is always the same
    meet(m, s, t);
    if (lane == 0) {
        sh.warp_stat[warp][0] = m;
        sh.warp_stat[warp][1] = s;
        sh.warp_stat[warp][2] = t;
    }
    __syncthreads();
    if (warp == 0) {
        m = lane < WARPS ? sh.warp_stat[lane][0] : -INFINITY;
        s = lane < WARPS ? sh.warp_stat[lane][1] : 0.0f;
        t = lane < WARPS ? sh.warp_stat[lane][2] : 0.0f;
        meet(m, s, t);
        if (lane == 0) {
            sh.stat[0] = m;
            sh.stat[1] = s;
            sh.stat[2] = t;
            sh.count = sh.groups = 0;
        }
    }
    __syncthreads();
    if (k > 0) {
        const int n = find_best<THREADS>(sh, base, ahead, end, first, chunks, span, groups, k);
        cut<THREADS>(sh, n, k);
    }
    if (blocks > 1) {
        cluster_sync();
        if (block == 0) {
            // the blocks' best together (k each, what is none of a block's behind all others: blocks * k <= 512), then the row's
            for (int i = threadIdx.x; i < blocks * kMaxTop; i += THREADS) {
                const int c = i / kMaxTop, j = i % kMaxTop;
                if (j >= k) continue;
                sh.value[c * k + j] = __uint_as_float(peer_u32(&sh.best_value[j], c));
                sh.id[c * k + j] = (int)peer_u32(&sh.best_id[j], c);
            }
            if (warp == 0) {
                m = lane < blocks ? __uint_as_float(peer_u32(&sh.stat[0], lane)) : -INFINITY;
                s = lane < blocks ? __uint_as_float(peer_u32(&sh.stat[1], lane)) : 0.0f;
                t = lane < blocks ? __uint_as_float(peer_u32(&sh.stat[2], lane)) : 0.0f;
                meet(m, s, t);
            }
            __syncthreads();
            if ((int)threadIdx.x < k) {            // (what is no entry has no rank of its own)
                sh.best_value[threadIdx.x] = -INFINITY;
                sh.best_id[threadIdx.x] = kNobody;
            }
            __syncthreads();
            if (k > 0) cut<THREADS>(sh, blocks * k, k);
            if (threadIdx.x == 0) {
                sh.stat[0] = m;
                sh.stat[1] = s;
                sh.stat[2] = t;
            }
        }
        cluster_sync();                            // no block leaves while a peer may still read its shared memory
        if (block != 0) return;
    } else {
        __syncthreads();
    }
    const float high = sh.stat[0], log_sum = logf(sh.stat[1]);
    if (threadIdx.x == 0) {
        logprob[r] = (given - high) - log_sum;
        entropy[r] = log_sum - sh.stat[2] / sh.stat[1];
    }
    if (warp != 0) return;
    int kept = 0;
    for (int i0 = 0; i0 < k; i0 += 32) {
        const int i = i0 + lane;
        const bool is = i < k && sh.best_id[i] != kNobody;
        if (is) {
            top_value[r * k + i] = (sh.best_value[i] - high) - log_sum;
            top_id[r * k + i] = sh.best_id[i];
        }
        kept += __popc(__ballot_sync(0xffffffffu, is));
    }
    // Fewer than k logits above -inf: those at -inf (or NaN) follow, by id.  All but fewer than k are of that kind, so they are found
    // within 2 k tokens.
    for (int i0 = 0; i0 < vocab && kept < k; i0 += 32) {
        const int i = i0 + lane;
        const bool is = i < vocab && !(row[i] > -INFINITY);
        const unsigned who = __ballot_sync(0xffffffffu, is);
        const int place = kept + __popc(who & ((1u << lane) - 1));
        if (is && place < k) {
            top_value[r * k + place] = (row[i] - high) - log_sum;
            top_id[r * k + place] = i;
        }
        kept += __popc(who);
    }
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

template <int THREADS>
int launch_rows(int rows, int vocab, int blocks, cudaStream_t stream, const float* logits, int64_t stride, const int* tokens,
                float* logprob, float* entropy, float* top_value, int* top_id, int top) {
    while (blocks > 1 && vocab <= (blocks / 2) * kEach * THREADS) blocks >>= 1;      // (a chunk for each)
    if ((int64_t)rows * blocks > 0x7fffffff) return TB_ERR_BAD_SIZE;
    const int part = ((vocab + blocks - 1) / blocks + 3) / 4 * 4;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * blocks));
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = (size_t)kSlots * kPackets * THREADS * sizeof(float4);
    config.stream = stream;
    // (with the list and the groups more than a kernel may have unasked: told once a device)
    static bool told[64];
    int device = 0;
    if (const cudaError_t err = cudaGetDevice(&device)) return (int)err;
    if (device < 0 || device >= 64 || !told[device]) {
        if (const cudaError_t err = cudaFuncSetAttribute(logprobs_kernel<THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                         (int)config.dynamicSmemBytes))
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
    const cudaError_t err = cudaLaunchKernelEx(&config, logprobs_kernel<THREADS>, logits, stride, tokens, logprob, entropy,
                                               top_value, top_id, vocab, top, blocks, part);
    return err == cudaSuccess ? tb_launch_status() : (int)err;
}

}  // namespace

TB_EXPORT int tb_token_logprobs(const float* logits, int64_t stride, const int* tokens, float* logprob, float* entropy,
                                float* top_value, int* top_id, int rows, int vocab, int top, cudaStream_t stream) {
    if (rows == 0) return 0;
    if (rows < 0 || vocab <= 0 || vocab > (1 << 30) || top < 0 || top > kMaxTop || top > vocab) return TB_ERR_BAD_SIZE;
    // Few rows: blocks of 1,024, as many a row as leave each a multiprocessor of its own; up to two rows a multiprocessor one of 512
    // each, beyond one of 256.  (128,256 logits, twenty alternatives, device time of blocks of 256 / 512 / 1,024 at their best split:
    // 64 rows 20.1 / 15.0 / 14.7 us, 256 rows 31.3 / 28.6 / 34.6, 1,536 rows 145 / 153 / 183.)
    const int64_t sms = sm_count();
    if (rows <= sms) {
        int blocks = kMaxBlocks;
        while (rows * blocks > sms) blocks >>= 1;
        return launch_rows<1024>(rows, vocab, blocks, stream, logits, stride, tokens, logprob, entropy, top_value, top_id, top);
    }
    if (rows <= 2 * sms)
        return launch_rows<512>(rows, vocab, 1, stream, logits, stride, tokens, logprob, entropy, top_value, top_id, top);
    return launch_rows<256>(rows, vocab, 1, stream, logits, stride, tokens, logprob, entropy, top_value, top_id, top);
}
