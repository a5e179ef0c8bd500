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
// part each); a block takes its part in chunks of sixteen logits a thread, in registers, the next chunk's loads under way
// meanwhile.  Many rows: blocks of 256 threads, four a multiprocessor, so that one row's beginning and end run under the
// others' loads; few rows: blocks of 1,024, one chunk each at a vocabulary of 128,256.  Of a chunk
//   * every thread adds its numbers to a maximum, S and T of its own (rescaled when its maximum rises), all in 32 bits;
//     they meet once, at the end, in a fixed order, so a row's numbers do not depend on the timing;
//   * a thread whose maximum exceeds the k-th best logit so far puts what exceeds it into a list in shared memory.  Once
//     the first chunk is done few do: k numbers for the second chunk, k / 2 for the third.  A list that grows is cut to its k
//     best (each entry's rank is the number of entries in front of it).
//   * where more threads exceed it than the list could hold (the first chunk, or logits that rise with the id) a bound comes
//     first: the k-th largest of 64 thread maxima (each warp's largest few), which k logits of the chunk reach.  Should more
//     threads reach that than fit, the interval of the maxima's bit patterns is halved until few enough do; and if equal
//     numbers leave no such bound, what lies above is taken and of the equal ones those of lowest id.
#include "common.cuh"

namespace {

constexpr int kPackets = 4;                        // 16-byte loads of a thread and chunk
constexpr int kEach = 4 * kPackets;                // logits of a thread and chunk
constexpr int kMaxTop = 64;
constexpr int kListed = 2048;                      // entries of the list
constexpr int kRoom = (kListed - kMaxTop) / kEach; // threads that may add to a list of at most kMaxTop entries (124)
static_assert(kRoom >= kMaxTop, "a bound that kMaxTop threads reach must fit");
constexpr int kCut = 96;                           // a list this much longer than k is cut after a chunk
constexpr int kMaxBlocks = 8;
constexpr int kNobody = 0x7fffffff;                // the id of an entry that is none
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1024.0f;                   // e^x is 0 in 32 bits from here on down

struct Shared {
    float value[kListed];
    int id[kListed];
    float best_value[kMaxTop];                     // k entries in order, behind those there are (-inf, kNobody)
    int best_id[kMaxTop];
    uint32_t sample[kMaxTop];                      // thread maxima, the largest of each warp
    float warp_stat[32][3];
    int warp_count[32];
    float stat[3];                                 // this block's m, S, T
    uint32_t bound;
    int count;                                     // entries of the list
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

// (m, S, T) of two disjoint sets of numbers
__device__ __forceinline__ void join(float& m, float& s, float& t, float m2, float s2, float t2) {
    const float top = fmaxf(m, m2);
    if (!(top > -INFINITY)) {                      // nothing in either (a NaN in s or t stays)
        s += s2;
        t += t2;
        return;
    }
    // (where e^(m - top) is 0, the distance must not make an infinity of what it is multiplied by; an infinite top gives NaN)
    const float a = exp2_of((m - top) * kLog2e), b = exp2_of((m2 - top) * kLog2e);
    const float da = fmaxf(m - top, kFar), db = fmaxf(m2 - top, kFar);
    t = (t + s * da) * a + (t2 + s2 * db) * b;
    s = s * a + s2 * b;
    m = top;
}
// The same over the first `count` (a power of two) lanes of a warp; every lane gets the result.
__device__ __forceinline__ void join_lanes(float& m, float& s, float& t, int count) {
    for (int o = 1; o < count; o <<= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        const float t2 = __shfl_xor_sync(0xffffffffu, t, o);
        join(m, s, t, m2, s2, t2);
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
// it.  `share` threads count for one entry.  Every thread calls this; the list is whole (a barrier in front).
template <int THREADS>
__device__ __forceinline__ void cut(Shared& sh, int n, int k) {
    int share = 1;
    while (share < 32 && n * share * 2 <= THREADS) share *= 2;
    if ((int)threadIdx.x >= n && (int)threadIdx.x < k) {
        sh.best_value[threadIdx.x] = -INFINITY;
        sh.best_id[threadIdx.x] = kNobody;
    }
    for (int base = 0; base < n; base += THREADS / share) {
        const int e = base + (int)threadIdx.x / share, part = (int)threadIdx.x % share;
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

// The list of n entries becomes the k best alone.  Returns the value that a later logit has to exceed.
template <int THREADS>
__device__ __forceinline__ float recut(Shared& sh, int n, int k) {
    const int kept = min(n, k);
    cut<THREADS>(sh, n, k);
    if ((int)threadIdx.x < kept) {
        sh.value[threadIdx.x] = sh.best_value[threadIdx.x];
        sh.id[threadIdx.x] = sh.best_id[threadIdx.x];
    }
    if (threadIdx.x == 0) sh.count = kept;
    const float bound = kept == k ? sh.best_value[k - 1] : -INFINITY;
    __syncthreads();
    return bound;
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

// grid: rows * blocks; the blocks of a row are one cluster.
template <int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
logprobs_kernel(const float* __restrict__ logits, int64_t stride, const int* __restrict__ tokens,
                float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_value,
                int* __restrict__ top_id, int vocab, int k, int blocks, int part) {
    constexpr int WARPS = THREADS / 32, kChunk = kEach * THREADS;
    constexpr int kSampled = kMaxTop / WARPS;      // thread maxima of a warp among the sample
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
    if (threadIdx.x == 0) sh.count = 0;
    pdl_wait();                                    // the logits come from the kernel in front
    float given = NAN;
    if (block == 0 && threadIdx.x == 0) {
        const int token = tokens[r];
        if (token >= 0 && token < vocab) given = row[token];
    }

    auto fetch = [&](float4 (&held)[kPackets], int chunk) {
#pragma unroll
        for (int u = 0; u < kPackets; ++u) {
            const int i = chunk + (u * THREADS + (int)threadIdx.x) * 4;
            if (i >= ahead && i + 4 <= end) {
                held[u] = __ldcs(reinterpret_cast<const float4*>(base + i));
            } else {
                held[u].x = i >= ahead && i < end ? base[i] : -INFINITY;
                held[u].y = i + 1 >= ahead && i + 1 < end ? base[i + 1] : -INFINITY;
                held[u].z = i + 2 >= ahead && i + 2 < end ? base[i + 2] : -INFINITY;
                held[u].w = i + 3 >= ahead && i + 3 < end ? base[i + 3] : -INFINITY;
            }
        }
    };

    float m = -INFINITY, s = 0.0f, t = 0.0f, bound = -INFINITY;
    int listed = 0;                                // entries of the list, as every thread knows them between two chunks
    float4 next[kPackets];
    fetch(next, 0);
    for (int chunk = 0; chunk < end; chunk += kChunk) {
        float x[kEach];
#pragma unroll
        for (int u = 0; u < kPackets; ++u) {
            x[4 * u] = next[u].x;
            x[4 * u + 1] = next[u].y;
            x[4 * u + 2] = next[u].z;
            x[4 * u + 3] = next[u].w;
        }
        if (chunk + kChunk < end) fetch(next, chunk + kChunk);
        float top = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
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
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float d = x[i] - low, e = exp2_of(d * kLog2e);
            s += e;
            t += fmaxf(d, kFar) * e;               // (-inf adds nothing, a NaN comes in by e)
        }
        if (k == 0) continue;
        auto id_of = [&](int i) { return first + chunk + ((i >> 2) * THREADS + (int)threadIdx.x) * 4 + (i & 3) - ahead; };
        auto add = [&](bool wanted, int i) {
            if (!wanted) return;
            const int at = atomicAdd(&sh.count, 1);
            sh.value[at] = x[i];
            sh.id[at] = id_of(i);
        };
        const int over = __syncthreads_count(top > bound);
        if (over == 0) continue;
        bool cut_now;
        if (over * kEach + listed <= kListed) {
            if (top > bound) {
#pragma unroll
                for (int i = 0; i < kEach; ++i) add(x[i] > bound, i);
            }
            cut_now = over >= k;
        } else {
            cut_now = true;
            if (listed > k) bound = recut<THREADS>(sh, listed, k);
            const uint32_t mine = ordered(top), floor = ordered(bound);
            // the sample: each warp's kSampled largest maxima (of different threads)
            uint32_t rest = mine, largest = 0;
#pragma unroll
            for (int j = 0; j < kSampled; ++j) {
                const uint32_t best = __reduce_max_sync(0xffffffffu, rest);
                if (j == 0) largest = best;
                if (lane == 0) sh.sample[warp * kSampled + j] = best;
                if (lane == __ffs(__ballot_sync(0xffffffffu, rest == best)) - 1) rest = 0;
            }
            __syncthreads();
            // its k-th largest (equal ones by their place, so that exactly one has every rank), which k threads at least reach
            if (threadIdx.x < kMaxTop) {
                const uint32_t v = sh.sample[threadIdx.x];
                int rank = 0;
#pragma unroll 8
                for (int j = 0; j < kMaxTop; ++j) {
                    const uint32_t o = sh.sample[j];
                    rank += o > v || (o == v && j < (int)threadIdx.x) ? 1 : 0;
                }
                if (rank == k - 1) sh.bound = v;
                if (rank == 0) sh.warp_count[0] = (int)v;           // the block's largest
            }
            __syncthreads();
            uint32_t low_key = max(sh.bound, floor + 1);
            largest = (uint32_t)sh.warp_count[0];
            int reach = __syncthreads_count(mine >= low_key);
            if (reach > kRoom) {
                // low_key: what at least k threads reach, or all that exceed the bound; high_key: what fewer than k reach
                uint32_t high_key = largest + 1;
                while (high_key > low_key + 1) {
                    const uint32_t middle = low_key + (high_key - low_key) / 2;
                    reach = __syncthreads_count(mine >= middle);
                    if (reach < k) {
                        high_key = middle;
                    } else {
                        low_key = middle;
                        if (reach <= kRoom) break;
                    }
                }
                reach = __syncthreads_count(mine >= low_key);
            }
            const float cutoff = from_ordered(low_key);
            if (reach <= kRoom) {
                if (mine >= low_key) {
#pragma unroll
                    for (int i = 0; i < kEach; ++i) add(x[i] >= cutoff && x[i] > bound, i);
                }
            } else {
                // more threads than fit have `cutoff` as their maximum, fewer than k a larger one: all that is larger, and of
                // what is equal to it the first k by id (packets of a lower u come first, then lower threads)
                if (top > cutoff) {
#pragma unroll
                    for (int i = 0; i < kEach; ++i) add(x[i] > cutoff, i);
                }
                int taken = 0;
                for (int u = 0; u < kPackets && taken < k; ++u) {
                    int equal = 0;
#pragma unroll
                    for (int i = 0; i < kEach; ++i) equal += (i >> 2) == u && x[i] == cutoff ? 1 : 0;
                    int all;
                    int at = taken + sum_before<THREADS>(sh, equal, all);
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        if ((i >> 2) == u && x[i] == cutoff) {
                            add(at < k, i);
                            ++at;
                        }
                    }
                    taken += all;
                }
            }
        }
        __syncthreads();
        listed = sh.count;                         // (nothing is added before the next chunk's barrier)
        if (cut_now || listed > k + kCut) {
            bound = recut<THREADS>(sh, listed, k);
            listed = min(listed, k);
        }
    }

    // the block's sums, in the order of lanes and warps
    join_lanes(m, s, t, 32);
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
        join_lanes(m, s, t, WARPS);
        if (lane == 0) {
            sh.stat[0] = m;
            sh.stat[1] = s;
            sh.stat[2] = t;
        }
    }
    if (k > 0) cut<THREADS>(sh, listed, k);
    if (blocks > 1) {
        cluster_sync();
        if (block == 0) {
            // the blocks' best together (k each, what is none of a block's behind all others: blocks * k <= 512), then the row's
            for (int i = threadIdx.x; i < blocks * k; i += THREADS) {
                sh.value[i] = __uint_as_float(peer_u32(&sh.best_value[i % k], i / k));
                sh.id[i] = (int)peer_u32(&sh.best_id[i % k], i / k);
            }
            if (warp == 0) {
                m = lane < blocks ? __uint_as_float(peer_u32(&sh.stat[0], lane)) : -INFINITY;
                s = lane < blocks ? __uint_as_float(peer_u32(&sh.stat[1], lane)) : 0.0f;
                t = lane < blocks ? __uint_as_float(peer_u32(&sh.stat[2], lane)) : 0.0f;
                join_lanes(m, s, t, kMaxBlocks);
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
    config.stream = stream;
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
    // few rows: large blocks, as many a row as keep one a multiprocessor; many: small ones, four a multiprocessor
    const int64_t sms = sm_count();
    if (rows * kMaxBlocks <= sms)
        return launch_rows<1024>(rows, vocab, kMaxBlocks, stream, logits, stride, tokens, logprob, entropy, top_value, top_id, top);
    int blocks = kMaxBlocks;
    while (blocks > 1 && (int64_t)rows * blocks > 4 * sms) blocks >>= 1;
    return launch_rows<256>(rows, vocab, blocks, stream, logits, stride, tokens, logprob, entropy, top_value, top_id, top);
}
