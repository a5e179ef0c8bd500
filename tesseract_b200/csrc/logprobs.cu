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
// part each); a block takes its part in chunks of 8,192 logits, sixteen a thread in registers, the next chunk's loads
// under way meanwhile.  Of a chunk
//   * every thread adds its numbers to a maximum, S and T of its own (rescaled when its maximum rises), all in 32 bits;
//     they meet once, at the end, in a fixed order, so a row's numbers do not depend on the timing;
//   * a thread whose maximum exceeds the k-th best logit so far puts what exceeds it into a list in shared memory.  Once
//     the first chunk is done few do: k numbers for the second chunk, k / 2 for the third.  A list that grows is cut to its k
//     best (each entry's rank is the number of entries in front of it).
//   * where more threads exceed it than the list could hold (the first chunk, or logits that rise with the id), a bound
//     that at least k threads' maxima reach is found first, by halving the interval of the maxima's bit patterns; if equal
//     numbers leave no bound that few enough reach, what lies above is taken and of the equal ones those of lowest id.
#include "common.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kPackets = 4;                        // 16-byte loads of a thread and chunk
constexpr int kEach = 4 * kPackets;                // logits of a thread and chunk
constexpr int kChunk = kEach * kThreads;
constexpr int kMaxTop = 64;
constexpr int kListed = 2048;                      // entries of the list
constexpr int kRoom = (kListed - kMaxTop) / kEach; // threads that may add to a list of at most kMaxTop entries (124)
static_assert(kRoom >= kMaxTop, "a bound that kMaxTop threads reach must fit");
constexpr int kCut = 96;                           // a list this much longer than k is cut after a chunk
constexpr int kMaxBlocks = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -1024.0f;                   // e^x is 0 in 32 bits from here on down

struct Shared {
    float value[kListed];
    int id[kListed];
    float best_value[kMaxTop];
    int best_id[kMaxTop];
    float warp_stat[kWarps][3];
    uint32_t warp_low[kWarps], warp_high[kWarps];
    int warp_count[kWarps];
    float stat[3];                                 // this block's m, S, T
    int count;                                     // entries of the list
    int kept;                                      // entries of best_*
};

// floats as unsigned numbers of the same order (-inf smallest; NaN never gets here)
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t u = __float_as_uint(v);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
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
    const float a = exp2f((m - top) * kLog2e), b = exp2f((m2 - top) * kLog2e);
    const float da = fmaxf(m - top, kFar), db = fmaxf(m2 - top, kFar);
    t = (t + s * da) * a + (t2 + s2 * db) * b;
    s = s * a + s2 * b;
    m = top;
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

// Cuts the list to its k best, in order, in best_value / best_id: the rank of an entry is the number of entries in front of
// it.  `share` threads count for one entry.  Every thread calls this; the list is whole (a barrier in front).
__device__ __forceinline__ void cut(Shared& sh, int n, int k) {
    int share = 1;
    while (share < 32 && n * share * 2 <= kThreads) share *= 2;
    for (int base = 0; base < n; base += kThreads / share) {
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
__device__ __forceinline__ float recut(Shared& sh, int n, int k) {
    const int kept = min(n, k);
    cut(sh, n, k);
    if ((int)threadIdx.x < kept) {
        sh.value[threadIdx.x] = sh.best_value[threadIdx.x];
        sh.id[threadIdx.x] = sh.best_id[threadIdx.x];
    }
    if (threadIdx.x == 0) sh.count = kept;
    const float bound = kept == k ? sh.best_value[k - 1] : -INFINITY;
    __syncthreads();
    return bound;
}

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
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sh.warp_count[w];
        all += sh.warp_count[w];
    }
    return before;
}

// grid: rows * blocks; the blocks of a row are one cluster.
__global__ void __launch_bounds__(kThreads, 2)
logprobs_kernel(const float* __restrict__ logits, int64_t stride, const int* __restrict__ tokens,
                float* __restrict__ logprob, float* __restrict__ entropy, float* __restrict__ top_value,
                int* __restrict__ top_id, int vocab, int k, int blocks, int part) {
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
    __syncthreads();
    pdl_wait();                                    // the logits come from the kernel in front
    float given = NAN;
    if (block == 0 && threadIdx.x == 0) {
        const int token = tokens[r];
        if (token >= 0 && token < vocab) given = row[token];
    }

    auto fetch = [&](float4 (&held)[kPackets], int chunk) {
#pragma unroll
        for (int u = 0; u < kPackets; ++u) {
            const int i = chunk + (u * kThreads + (int)threadIdx.x) * 4;
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
                const float d = m - top, a = exp2f(d * kLog2e);
                t = (t + s * fmaxf(d, kFar)) * a;
                s *= a;
            }
            m = top;
        }
        const float low = m > -INFINITY ? m : 0.0f;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float d = x[i] - low, e = exp2f(d * kLog2e);
            s += e;
            t += fmaxf(d, kFar) * e;               // (-inf adds nothing, a NaN comes in by e)
        }
        if (k == 0) continue;
        auto id_of = [&](int i) { return first + chunk + ((i >> 2) * kThreads + (int)threadIdx.x) * 4 + (i & 3) - ahead; };
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
            if (listed > k) bound = recut(sh, listed, k);
            // a bound that at least k and at most kRoom threads' maxima reach
            const uint32_t mine = ordered(top), floor = ordered(bound);
            uint32_t smallest = __reduce_min_sync(0xffffffffu, mine), largest = __reduce_max_sync(0xffffffffu, mine);
            if (lane == 0) {
                sh.warp_low[warp] = smallest;
                sh.warp_high[warp] = largest;
            }
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                smallest = min(smallest, sh.warp_low[w]);
                largest = max(largest, sh.warp_high[w]);
            }
            // low_key: what at least k threads reach, or all that exceed the bound; high_key: what fewer than k reach
            uint32_t low_key = max(smallest, floor + 1), high_key = largest + 1;
            int reach;
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
                    int at = taken + sum_before(sh, equal, all);
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
            bound = recut(sh, listed, k);
            listed = min(listed, k);
        }
    }

    // the block's sums, in the order of lanes and warps
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
        const float t2 = __shfl_xor_sync(0xffffffffu, t, o);
        join(m, s, t, m2, s2, t2);
    }
    if (lane == 0) {
        sh.warp_stat[warp][0] = m;
        sh.warp_stat[warp][1] = s;
        sh.warp_stat[warp][2] = t;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kWarps; ++w) join(m, s, t, sh.warp_stat[w][0], sh.warp_stat[w][1], sh.warp_stat[w][2]);
        sh.stat[0] = m;
        sh.stat[1] = s;
        sh.stat[2] = t;
    }
    if (k > 0) {
        cut(sh, listed, k);
        if (threadIdx.x == 0) sh.kept = min(listed, k);
    }
    if (blocks > 1) {
        cluster_sync();
        if (block == 0) {
            if (threadIdx.x == 0) {
                m = sh.stat[0], s = sh.stat[1], t = sh.stat[2];
                for (int c = 1; c < blocks; ++c)
                    join(m, s, t, __uint_as_float(peer_u32(&sh.stat[0], c)), __uint_as_float(peer_u32(&sh.stat[1], c)),
                         __uint_as_float(peer_u32(&sh.stat[2], c)));
            }
            if (k > 0) {
                // the blocks' best together (each at most k: blocks * k <= kListed), then the row's
                int n = 0;
                for (int c = 0; c < blocks; ++c) {
                    const int kept = (int)peer_u32(&sh.kept, c);
                    for (int i = threadIdx.x; i < kept; i += kThreads) {
                        sh.value[n + i] = __uint_as_float(peer_u32(&sh.best_value[i], c));
                        sh.id[n + i] = (int)peer_u32(&sh.best_id[i], c);
                    }
                    n += kept;
                }
                __syncthreads();
                cut(sh, n, k);
                if (threadIdx.x == 0) sh.kept = min(n, k);
            }
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
    const int kept = k > 0 ? sh.kept : 0;
    for (int i = threadIdx.x; i < kept; i += kThreads) {
        top_value[r * k + i] = (sh.best_value[i] - high) - log_sum;
        top_id[r * k + i] = sh.best_id[i];
    }
    if (kept < k && warp == 0) {
        // fewer than k logits above -inf: those at -inf (or NaN) follow, by id.  All but fewer than k are of that kind, so the
        // first warp finds them within 2 k tokens.
        int at = kept;
        for (int i0 = 0; i0 < vocab && at < k; i0 += 32) {
            const int i = i0 + lane;
            const bool is = i < vocab && !(row[i] > -INFINITY);
            const unsigned who = __ballot_sync(0xffffffffu, is);
            const int place = at + __popc(who & ((1u << lane) - 1));
            if (is && place < k) {
                top_value[r * k + place] = (row[i] - high) - log_sum;
                top_id[r * k + place] = i;
            }
            at += __popc(who);
        }
    }
}

// Blocks of a row: as many (up to the portable cluster size) as keep the grid within the two blocks a multiprocessor that fit,
// and a chunk for each.
int blocks_per_row(int rows, int vocab) {
    static int sms = 0;
    if (sms == 0) {
        int device = 0;
        cudaGetDevice(&device);
        if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || sms <= 0) sms = 1;
    }
    int blocks = kMaxBlocks;
    while (blocks > 1 && ((int64_t)rows * blocks > 2 * sms || vocab <= (blocks / 2) * kChunk)) blocks >>= 1;
    return blocks;
}

}  // namespace

TB_EXPORT int tb_token_logprobs(const float* logits, int64_t stride, const int* tokens, float* logprob, float* entropy,
                                float* top_value, int* top_id, int rows, int vocab, int top, cudaStream_t stream) {
    if (rows == 0) return 0;
    if (rows < 0 || vocab <= 0 || vocab > (1 << 30) || top < 0 || top > kMaxTop || top > vocab) return TB_ERR_BAD_SIZE;
    const int blocks = blocks_per_row(rows, vocab);
    if ((int64_t)rows * blocks > 0x7fffffff) return TB_ERR_BAD_SIZE;
    const int part = ((vocab + blocks - 1) / blocks + 3) / 4 * 4;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(rows * blocks));
    config.blockDim = dim3(kThreads);
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
    const cudaError_t err = cudaLaunchKernelEx(&config, logprobs_kernel, logits, stride, tokens, logprob, entropy, top_value,
                                               top_id, vocab, top, blocks, part);
    return err == cudaSuccess ? tb_launch_status() : (int)err;
}
