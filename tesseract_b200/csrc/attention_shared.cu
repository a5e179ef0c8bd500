// Decoded rows over paged keys and values, where groups of rows have their first keys in common: those are read once for
// the whole group instead of once a row.
//
// Per row b and head h over the keys 0..p_b of the row (p_b: its position; -1: none), c = h / fold the kv head:
//   s_j = scale * q_bh . k_cj     o = sum_j 2^(s_j log2 e - m) v_cj / sum_j 2^(s_j log2 e - m)      (no key: 0)
// The keys are cut into the part that the row's group has in common, [0, L), L a multiple of 64, and the part behind,
// [L, p_b].  A softmax over disjoint parts is put together from their maxima m, sums l and unnormalised sums a of values,
// all kept in 32 bits:  m = max m_i,  l = sum l_i 2^(m_i - m),  o = sum a_i 2^(m_i - m) / l.  Both parts are cut further
// into runs of keys, so that few rows fill the chip; every run leaves (m, l, a) per row and head in scratch memory and a second
// kernel puts them together in the order of the runs (no atomics: the same call gives the same bits).
//
// What a block does: one tile of folded rows (the `fold` query heads of a kv head, row after row of the group, or of one row
// behind the common part) against one run of keys of one kv head.
//   attend_mma   bfloat16, tiles of 16 folded rows: the warps take turns at tiles of 16 keys, each through a cp.async ring of its
//                own into mma.sync.m16n8k16; scores and sums in 32 bits, the weights rounded to bfloat16 for their product with the
//                values (as in this package's other attention kernels in bfloat16: relative 2^-9 of each, averaged over the keys).
//                Bound by HBM: 16 rows of 4,000 keys of their own, 32 heads on 8 of 128, 262 MB in 47.3 us = 5.5 TB/s, 0.86 of the
//                measured copy rate; below some 10 MB by the chain of a launch, its look-ups and the first copies (4 to 12 us).
//   attend_tc    bfloat16, common parts of groups with more folded rows: tiles of 128 on the tcgen05 tensor
//                cores, see there.  A tile of 16 would read a common part from L2 once for every 16 folded rows.
//   attend_f32, attend_f32_wide   32-bit, tiles of 8 and of 32 folded rows, multiply-adds only, see there.
// Which form and how many runs: plan.shared_attention, with both sides' times beside its rule.
// What rounding the weights costs: against 64 bits a result is off by 0.0018 of its size in attend_mma and by up to 0.0023 in
// attend_tc, whose weights are seldom taken against their own maximum (which rounds without an error); 0.0017 of both is the
// result's own rounding.  In 32 bits it is 3e-7.
// Keys beyond a run's end are filled with zeros on the way in and masked, so whatever lies behind a row's last key in its page
// (numbers of an earlier owner, NaN) reaches nothing.
#include <cstring>
#include <new>
#include <set>

#include "tma.cuh"

namespace {

using namespace tbtma;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kMasked = -1.0e30f;
constexpr int kBlock = 64;                    // keys that common parts and runs are counted in

struct SharedParams {
    const void* q;                            // [rows, heads * head_dim], row stride q_stride
    void* out;
    const void* cache;                        // [page][K|V][kv head][page_size][head_dim]
    const int* positions;                     // [rows]
    const int* table;                         // [rows, table_stride]
    const int* members;                       // [rows]: the rows group by group
    const int* group_start;                   // [groups + 1]: where a group's rows begin in `members`
    const int* leader;                        // [groups]: the row through whose table the keys in common are read
    const int* prefix;                        // [groups]: keys in common (whole blocks; 0 for a row alone)
    const int* common;                        // [rows]: those of the row's group
    float* part_a;                            // [rows][heads][parts][head_dim]
    float2* part_ml;                          // [rows][heads][parts]
    int64_t q_stride, out_stride;
    int table_stride, table_keys;             // keys that a row of the table can name
    int rows, groups, heads, kv_heads, fold, head_dim;
    int tiles;                                // tiles of all groups' folded rows
    int prefix_parts, prefix_run;             // runs of a common part: at most so many, of at least so many blocks of keys each
    int tail_parts, tail_run;                 // the same behind it
    Paging paging;
    float scale_log2;
    int wide;                                 // the common parts are a kernel's of their own (attend_tc, attend_f32_wide)
    int direct;                               // one run a row and nothing in common: the results go to `out` at once
    int* error;                               // set where a bounded wait ran out
};

// One block's work.
struct Work {
    int first_member, member_rows;            // the tile's rows: `members[first_member ..]`, or (member_rows 0) the one row `row`
    int row;                                  // a row whose table names the keys
    int folded, first_folded;                 // folded rows of the group or row, and the first of the tile
    int kv_head, begin, end;                  // keys [begin, end)
    int part;                                 // slot of the partial result
};

// Keys in common as the kernel takes them: none where nothing is shared, and no more than a table can name.
__device__ __forceinline__ int common_keys(const SharedParams& p, int keys) {
    return p.prefix_parts == 0 ? 0 : min(keys, p.table_keys) & ~(kBlock - 1);
}

// How `blocks` blocks of keys are cut: runs of the same number of blocks, at most `parts`.  Returns the blocks of a run.
__device__ __forceinline__ int run_blocks(int blocks, int parts, int run) {
    const int n = min(parts, (blocks + run - 1) / run);
    return (blocks + n - 1) / n;
}

__device__ __forceinline__ int64_t common_blocks(const SharedParams& p) { return (int64_t)p.tiles * p.kv_heads * p.prefix_parts; }

// The work of block `index` of those for the common parts (TILE folded rows a tile); false if there is none.  Heads go fastest,
// first runs come first: short parts have no later ones, and the blocks that find nothing to do are the last to start.
template <int TILE>
__device__ bool find_common(const SharedParams& p, int64_t index, Work& w) {
    w.kv_head = (int)(index % p.kv_heads);
    const int rest = (int)(index / p.kv_heads), part = rest / p.tiles;
    int tile = rest % p.tiles;
    // which group: a warp counts the tiles of 32 groups at a time (all that is known of a group is loaded at once)
    const int lane = threadIdx.x & 31;
    for (int base = 0; base < p.groups; base += 32) {
        const int g = base + lane;
        int start = 0, n = 0, keys = 0, leader = 0, mine = 0;
        if (g < p.groups) {
            start = p.group_start[g];
            n = p.group_start[g + 1] - start;
            keys = common_keys(p, p.prefix[g]);
            leader = p.leader[g];
            if (keys > 0) mine = (n * p.fold + TILE - 1) / TILE;
        }
        int up_to = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, up_to, o);
            if (lane >= o) up_to += other;
        }
        const unsigned past = __ballot_sync(0xffffffffu, up_to > tile);
        if (past == 0) {
            tile -= __shfl_sync(0xffffffffu, up_to, 31);
            continue;
        }
        const int who = __ffs(past) - 1;
        tile -= __shfl_sync(0xffffffffu, up_to - mine, who);
        const int blocks = __shfl_sync(0xffffffffu, keys, who) / kBlock;
        const int run = run_blocks(blocks, p.prefix_parts, p.prefix_run);
        w.begin = part * run * kBlock;
        w.end = min(blocks, (part + 1) * run) * kBlock;
        w.first_member = __shfl_sync(0xffffffffu, start, who);
        w.member_rows = __shfl_sync(0xffffffffu, n, who);
        w.row = __shfl_sync(0xffffffffu, leader, who);
        w.folded = w.member_rows * p.fold;
        w.first_folded = tile * TILE;
        w.part = part;
        return w.begin < w.end;
    }
    return false;
}

// The work of block `index` of those for the keys behind, row by row.
template <int TILE>
__device__ bool find_tail(const SharedParams& p, int64_t index, Work& w) {
    w.kv_head = (int)(index % p.kv_heads);
    const int tiles = (p.fold + TILE - 1) / TILE;
    int rest = (int)(index / p.kv_heads);
    w.first_folded = rest % tiles * TILE;
    rest /= tiles;
    w.row = rest % p.rows;
    w.member_rows = 0;
    w.folded = p.fold;
    const int part = rest / p.rows;
    if (part >= p.tail_parts) return false;
    const int first = common_keys(p, p.common[w.row]);
    const int last = min(p.positions[w.row] + 1, p.table_keys);
    if (last <= first) return false;
    const int blocks = (last - first + kBlock - 1) / kBlock;
    const int run = run_blocks(blocks, p.tail_parts, p.tail_run);
    w.begin = first + part * run * kBlock;
    w.end = min(last, w.begin + run * kBlock);
    if (w.begin >= w.end) return false;
    w.part = p.prefix_parts + part;
    return true;
}

template <int TILE>
__device__ __forceinline__ bool find_work(const SharedParams& p, int64_t index, Work& w) {
    const int64_t common = common_blocks(p);
    return index < common ? find_common<TILE>(p, index, w) : find_tail<TILE>(p, index - common, w);
}

// Row of the batch and head of folded row `fr`.
__device__ __forceinline__ void place_of(const SharedParams& p, const Work& w, int fr, int& row, int& head) {
    const int member = fr / p.fold;
    row = w.member_rows > 0 ? p.members[w.first_member + member] : w.row;
    head = w.kv_head * p.fold + (fr - member * p.fold);
}

__device__ __forceinline__ int64_t slot_of(const SharedParams& p, int row, int head, int part) {
    return ((int64_t)row * p.heads + head) * (p.prefix_parts + p.tail_parts) + part;
}

// Waits, with a limit, for copies that are under way when something has been given up.
__device__ __noinline__ void settle(uint32_t bar, uint32_t parity) {
    for (uint32_t spin = 0; spin < kSpinLimit && !mbar_try_wait(bar, parity); ++spin) {
    }
}

template <typename T>
__device__ __forceinline__ void store_out(const SharedParams& p, int row, int head, int col, float v) {
    Elem<T>::store((T*)p.out + (int64_t)row * p.out_stride + (int64_t)head * p.head_dim + col, v);
}

// The warps' results of a tile, (m, l) in `ml` [warps][TILE][2] and sums in `acc` [warps][TILE][PITCH], put together in the
// order of the warps and left as the run's.  Every warp has written its own (a barrier in front).
template <typename T, int TILE, int PITCH, int WARPS>
__device__ void leave_run(const SharedParams& p, const Work& w, const float* ml, const float* acc) {
    const int rows = min(TILE, w.folded - w.first_folded);
    for (int idx = threadIdx.x; idx < rows * p.head_dim; idx += WARPS * 32) {
        const int r = idx / p.head_dim, col = idx - r * p.head_dim;
        float big = kMasked;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) big = fmaxf(big, ml[(v * TILE + r) * 2]);
        float a = 0.0f, l = 0.0f;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) {
            const float weight = exp2f(ml[(v * TILE + r) * 2] - big);
            a += weight * acc[(v * TILE + r) * PITCH + col];
            l += weight * ml[(v * TILE + r) * 2 + 1];
        }
        int row, head;
        place_of(p, w, w.first_folded + r, row, head);
        if (p.direct) {
            store_out<T>(p, row, head, col, a / l);
            continue;
        }
        const int64_t slot = slot_of(p, row, head, w.part);
        p.part_a[slot * p.head_dim + col] = a;
        if (col == 0) p.part_ml[slot] = make_float2(big, l);
    }
}

// The zeros of a row without keys, where nothing behind this kernel writes them.
template <typename T, int TILE>
__device__ void leave_nothing(const SharedParams& p, const Work& w) {
    const int rows = min(TILE, w.folded - w.first_folded);
    for (int idx = threadIdx.x; idx < rows * p.head_dim; idx += blockDim.x) {
        const int r = idx / p.head_dim;
        store_out<T>(p, w.row, w.kv_head * p.fold + w.first_folded + r, idx - r * p.head_dim, 0.0f);
    }
}

// ------------------------------------------------------------------------------------------------ bfloat16, mma.sync

constexpr int kKeys = 16;                     // keys of a warp's tile
constexpr int kRows = 16;                     // folded rows of a block's tile
// Warps and ring depth so that two blocks share a multiprocessor up to a padded head size of 128; blocks of two warps: eight, or four of
// a head size of 128 (deeper rings: 16 rows of 4,000 keys, 32 heads of 128, 56.8 us with two stages and six blocks a multiprocessor).
template <int D>
constexpr int kWarps = D <= 64 ? 8 : D <= 128 ? 6 : 4;
template <int D, int WARPS>
constexpr int kStages = D > 64 && D <= 128 && WARPS > 2 ? 2 : 3;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    const int bytes = valid ? 16 : 0;         // (0: the destination is filled with zeros)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x) {      // 2^x, relative error about 2^-22
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}
// Byte offset of 16-byte chunk `chunk` of row `row` in a [rows][D] tile, permuted so that the eight rows which an ldmatrix reads lie
// on different banks.
template <int D>
__device__ __forceinline__ uint32_t tile_offset(int row, int chunk) {
    constexpr int CH = D / 8;
    const int key = CH >= 8 ? (row & 7) : ((row >> 1) & (CH - 1));
    return (uint32_t)(row * (D * 2) + ((chunk ^ key) << 4));
}

template <int D, int WARPS, bool ONE>
__device__ void attend_mma(const SharedParams& p, const Work& w, unsigned char* smem) {
    constexpr int STAGES = kStages<D, WARPS>, CH = D / 8, PASSES = kKeys * CH / 32, LOOKS = ONE ? 1 : PASSES;
    constexpr uint32_t kTileBytes = kKeys * D * 2, kStageBytes = 2 * kTileBytes;
    constexpr bool QREG = D <= 128;           // the queries' fragments stay in registers
    constexpr int PITCH = D + 8;              // floats between rows of the sums that are put together (bank conflicts)
    static_assert((kKeys * CH) % 32 == 0, "a warp copies whole passes of 32 chunks");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = min(kRows, w.folded - w.first_folded);
    const uint32_t q_tile = smem_u32(smem);
    const uint32_t ring = q_tile + kRows * D * 2 + warp * (STAGES * kStageBytes);
    const __nv_bfloat16* q = (const __nv_bfloat16*)p.q;
    for (int idx = threadIdx.x; idx < kRows * CH; idx += WARPS * 32) {
        const int r = idx / CH, c = idx % CH;
        const bool ok = r < rows && c * 8 < p.head_dim;
        const __nv_bfloat16* src = q;
        if (ok) {
            int row, head;
            place_of(p, w, w.first_folded + r, row, head);
            src = q + (int64_t)row * p.q_stride + (int64_t)head * p.head_dim + c * 8;
        }
        cp_async16(q_tile + tile_offset<D>(r, c), src, ok);
    }
    const int* table = p.table + (int64_t)w.row * p.table_stride;
    const int64_t head_block = (int64_t)p.paging.size * p.head_dim;
    const int64_t page_block = 2 * (int64_t)p.kv_heads * head_block, v_offset = (int64_t)p.kv_heads * head_block;
    const __nv_bfloat16* base = (const __nv_bfloat16*)p.cache + (int64_t)w.kv_head * head_block;
    // The page of a tile's keys is looked up one tile ahead of the copies, which depend on it.  Runs begin with a block, so with pages
    // of a multiple of 16 keys a tile lies in one page, its keys one behind the other; otherwise (ONE false) every key has its own.
    auto look_up = [&](int key0, int (&pages)[LOOKS]) {
#pragma unroll
        for (int pass = 0; pass < LOOKS; ++pass) {
            const int key = ONE ? key0 : key0 + (pass * 32 + lane) / CH;
            pages[pass] = key < w.end ? table[p.paging.page_of(key)] : 0;
        }
    };
    auto bring = [&](uint32_t dst, int key0, const int (&pages)[LOOKS]) {
        const __nv_bfloat16* tile = nullptr;
        if (ONE) tile = base + (int64_t)pages[0] * page_block + (int64_t)p.paging.within(key0) * p.head_dim;
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) {
            const int idx = pass * 32 + lane, r = idx / CH, c = idx % CH, key = key0 + r;
            const bool ok = key < w.end && c * 8 < p.head_dim;
            const __nv_bfloat16* src = base;
            if (ONE) src = ok ? tile + r * p.head_dim + c * 8 : base;
            else if (ok) src = base + (int64_t)pages[pass % LOOKS] * page_block + (int64_t)p.paging.within(key) * p.head_dim + c * 8;
            const uint32_t offset = tile_offset<D>(r, c);
            cp_async16(dst + offset, src, ok);
            cp_async16(dst + kTileBytes + offset, src + v_offset, ok);
        }
    };
    int next_pages[LOOKS];
    int load_key = w.begin + warp * kKeys;
    constexpr int STEP = WARPS * kKeys;
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) {
        if (load_key < w.end) {
            look_up(load_key, next_pages);
            bring(ring + st * kStageBytes, load_key, next_pages);
        }
        cp_async_commit();                    // one group a stage, empty or not; the first holds the queries too
        load_key += STEP;
    }
    if (load_key < w.end) look_up(load_key, next_pages);
    cp_async_wait<STAGES - 2>();
    __syncthreads();                          // the queries are there
    uint32_t qf[QREG ? D / 16 : 1][4];
    if (QREG) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) ldmatrix_x4(qf[ks], q_tile + tile_offset<D>(lane & 15, ks * 2 + (lane >> 4)));
    }
    float o[D / 8][4], m[2] = {kMasked, kMasked}, l[2] = {0.0f, 0.0f};
#pragma unroll
    for (int dt = 0; dt < D / 8; ++dt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][e] = 0.0f;

    int it = 0;
    for (int key0 = w.begin + warp * kKeys; key0 < w.end; key0 += STEP, ++it) {
        if (load_key < w.end) bring(ring + ((it + STAGES - 1) % STAGES) * kStageBytes, load_key, next_pages);
        cp_async_commit();
        load_key += STEP;
        if (load_key < w.end) look_up(load_key, next_pages);
        cp_async_wait<STAGES - 1>();
        __syncwarp();
        const uint32_t k_tile = ring + (it % STAGES) * kStageBytes, v_tile = k_tile + kTileBytes;
        float s[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            uint32_t a[4], b[4];
            if (QREG) {
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = qf[ks][e];
            } else {
                ldmatrix_x4(a, q_tile + tile_offset<D>(lane & 15, ks * 2 + (lane >> 4)));
            }
            ldmatrix_x4(b, k_tile + tile_offset<D>((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)));
            mma_bf16(s[0], a, b[0], b[1]);
            mma_bf16(s[1], a, b[2], b[3]);
        }
        // this thread's scores: rows lane / 4 and lane / 4 + 8, keys 2 (lane % 4), + 1, + 8, + 9
        const bool whole = key0 + kKeys <= w.end;
        float high[2] = {kMasked, kMasked};
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[nt][e] *= p.scale_log2;
                if (!whole && key0 + nt * 8 + 2 * (lane & 3) + (e & 1) >= w.end) s[nt][e] = -INFINITY;      // 2^(that - m) is 0
                high[e >> 1] = fmaxf(high[e >> 1], s[nt][e]);
            }
        float correction[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], 1));
            high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], 2));
            const float m_new = fmaxf(m[i], high[i]);
            correction[i] = fast_exp2(m[i] - m_new);
            m[i] = m_new;
            l[i] *= correction[i];
        }
#pragma unroll
        for (int dt = 0; dt < D / 8; ++dt) {
            o[dt][0] *= correction[0];
            o[dt][1] *= correction[0];
            o[dt][2] *= correction[1];
            o[dt][3] *= correction[1];
        }
        uint32_t weights[4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            float e4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                e4[e] = fast_exp2(s[nt][e] - m[e >> 1]);
                l[e >> 1] += e4[e];
            }
            weights[2 * nt] = pack_bf16(e4[0], e4[1]);
            weights[2 * nt + 1] = pack_bf16(e4[2], e4[3]);
        }
#pragma unroll
        for (int dp = 0; dp < D / 16; ++dp) {
            uint32_t b[4];
            ldmatrix_x4_trans(b, v_tile + tile_offset<D>((lane & 7) + (((lane >> 3) & 1) << 3), dp * 2 + (lane >> 4)));
            mma_bf16(o[2 * dp], weights, b[0], b[1]);
            mma_bf16(o[2 * dp + 1], weights, b[2], b[3]);
        }
        __syncwarp();                         // every lane is done with this stage before it is filled again
    }
    cp_async_wait<0>();
    __syncthreads();                          // the rings become the place where the warps' results meet
    float* ml = reinterpret_cast<float*>(smem);
    float* acc = ml + WARPS * kRows * 2;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int r = (lane >> 2) + i * 8;
        if ((lane & 3) == 0) {
            ml[(warp * kRows + r) * 2] = m[i];
            ml[(warp * kRows + r) * 2 + 1] = l[i];
        }
#pragma unroll
        for (int dt = 0; dt < D / 8; ++dt)
            *reinterpret_cast<float2*>(acc + (warp * kRows + r) * PITCH + dt * 8 + 2 * (lane & 3)) =
                make_float2(o[dt][2 * i], o[dt][2 * i + 1]);
    }
    __syncthreads();
    leave_run<__nv_bfloat16, kRows, PITCH, WARPS>(p, w, ml, acc);
}

template <int D, int WARPS, bool ONE>
__global__ void __launch_bounds__(WARPS * 32) shared_mma_kernel(const SharedParams p) {
    extern __shared__ __align__(128) unsigned char smem[];
    pdl_wait();
    pdl_trigger();                            // (only now: the kernels behind read what is older than this one without a wait of their own)
    Work w;
    // (wide: the common parts are the next kernel's)
    if (p.wide ? find_tail<kRows>(p, blockIdx.x, w) : find_work<kRows>(p, blockIdx.x, w)) attend_mma<D, WARPS, ONE>(p, w, smem);
    else if (p.direct) leave_nothing<__nv_bfloat16, kRows>(p, w);
}

template <int D, int WARPS>
constexpr size_t mma_bytes() {
    constexpr size_t tiles = (size_t)kRows * D * 2 + (size_t)WARPS * kStages<D, WARPS> * 2 * kKeys * D * 2;
    constexpr size_t meet = (size_t)WARPS * kRows * (2 + D + 8) * sizeof(float);
    return tiles > meet ? tiles : meet;
}

// ------------------------------------------------------------------------------------------------ bfloat16, tcgen05

// Common parts of groups with more than a few folded rows, head sizes up to 64, 128 and 256: a tile of 128 folded rows against a run
// of blocks of 64 keys.  (Head sizes between are filled up with zeros, 80 for one: 20 heads on 4, 64 rows at 32,768 keys 45 us, 338
// with tiles of 16; 8 heads on 2 of 256 45 and 365.)  Per block S = Q . K^T (tcgen05.mma, M128 x N64, both operands in shared memory
// as 64-number slices with the 128-byte swizzle, S in 64 columns of tensor memory), the weights 2^(s - m) of a row by the thread
// that owns it, rounded to bfloat16 into one of two buffers in tensor memory, and O += P . V (M128 x N D x K64, P from tensor
// memory), O in D columns.  No block needs a mask: a common part ends with a block, and what is beyond it belongs to the rows' own
// parts.
// Warps 0-3: softmax, a thread a row (warps whose rows do not exist leave at once); one lane of warp 4 issues the products for the
// scores and one lane of warp 6 those with the values; warp 5 brings keys and values, page by page, with cp.async.bulk.tensor into
// rings of their own.  All waits are bounded.
// 64 rows, 32 heads on 8 of 128, 32,768 keys in common: 48.4 us with the join behind it (134 MB, 20.8 us at the measured copy rate;
// 34 GFLOP, 20.2 us at the measured matrix rate).  A block of 64 keys takes a softmax warp some 2,080 cycles, two blocks of threads a
// multiprocessor: 1,050 for the weights (both blocks' exponentials are 1,024 of the special-function unit), 570 waiting for scores
// (two tiles read the same keys through L2, 8.6 TB/s), 160 for a buffer of weights, the rest on the way to and from tensor memory.
// Tried: two tiles in one block of threads with 512 columns (68.1 us), two threads a row (1.3 longer), both products' issue by one lane
// (53.3), a part of the exponentials on the multiply-add pipe (51.7; head size 64 71 instead of 66), queries in tensor memory (no
// change; with the weights in the scores' place, as head size 128 needs then, 56.7), all keys found in L2 (47.7).
constexpr int kTcRows = 128;
constexpr int kTcThreads = 224;
template <int D>
constexpr int kTcStages = D == 64 ? 4 : 2;    // of the keys' ring and of the values': 128 KB a multiprocessor (a third for keys of 128 changes nothing)
template <int D>
constexpr int kTcBlocks = D == 256 ? 1 : 2;   // that share a multiprocessor
template <int D>
struct TcShape {
    static constexpr uint32_t kColumns = D == 256 ? 512 : 256;    // of tensor memory: S 64, O D, two buffers of P of 32
    static constexpr uint32_t kSlice = kBlock * 128;              // 64 keys x 64 numbers
    static constexpr uint32_t kBlockBytes = (D / 64) * kSlice;    // a block of keys, or of values
    static constexpr uint32_t kQSlice = kTcRows * 128, kQBytes = (D / 64) * kQSlice;
    static constexpr size_t kBytes = (size_t)kQBytes + (size_t)2 * kTcStages<D> * kBlockBytes;
};

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return (uint32_t)(row * 128 + ((chunk ^ (row & 7)) << 4)); }
// a tile of 128-byte rows with the 128-byte swizzle, 1024 bytes between groups of eight rows
__device__ __forceinline__ uint64_t desc_sw128(uint32_t smem_addr, uint32_t lbo) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)lbo << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// D = F32, A = B = BF16; b_mn: B is MN-major
__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n, int b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load_32(uint32_t taddr, uint32_t (&r)[32]) {      // (tmem_wait_ld before the registers are used)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_store_16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
          "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
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

template <int D>
__device__ void attend_tc(const SharedParams& p, const Work& w, const CUtensorMap* cache_map, unsigned char* smem) {
    using Tiles = TcShape<D>;
    constexpr int STAGES = kTcStages<D>;
    constexpr uint32_t kSlice = Tiles::kSlice, kBlockBytes = Tiles::kBlockBytes;
    // k_full, k_empty, v_full, v_empty [STAGES] each, s_full, s_free, p_ready[2], o_full[2] (of block j: those of j & 1)
    __shared__ __align__(8) uint64_t bars[4 * STAGES + 6];
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile int abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int dim = p.head_dim;               // (queries and, by the tensor map, keys and values are zeros from there up to D)
    const int rows = min(kTcRows, w.folded - w.first_folded);
    const int live_threads = (rows + 31) / 32 * 32;               // of the softmax warps: those with a row
    const int n_blocks = (w.end - w.begin) / kBlock;
    const int* table = p.table + (int64_t)w.row * p.table_stride;
    const uint32_t q_tile = smem_u32(smem), key_tiles = q_tile + Tiles::kQBytes, value_tiles = key_tiles + STAGES * kBlockBytes;
    const uint32_t k_full = smem_u32(&bars[0]), k_empty = k_full + 8 * STAGES;
    const uint32_t v_full = k_empty + 8 * STAGES, v_empty = v_full + 8 * STAGES;
    const uint32_t s_full = v_empty + 8 * STAGES, s_free = s_full + 8;
    auto p_ready = [&](int j) { return s_full + 16 + 8 * (j & 1); };
    auto o_full = [&](int j) { return s_full + 32 + 8 * (j & 1); };
    auto phase = [&](int j) { return (uint32_t)(j >> 1) & 1u; };
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < 4 * STAGES; ++s) mbar_init(k_full + 8 * s, 1);
        mbar_init(s_full, 1);
        mbar_init(s_free, live_threads);
        for (int b = 0; b < 2; ++b) {
            mbar_init(p_ready(b), live_threads);
            mbar_init(o_full(b), 1);
        }
        mbar_fence_init();
    }
    if (warp == 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_base_slot)), "r"(Tiles::kColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // where a thread's query lies, and the page of a lane's keys in the first block: looked up while the rest is set up
    const int rows_per_copy = min(p.paging.size, kBlock), copies = kBlock / rows_per_copy;          // keys and copies of a block: at most 8
    int row = 0, head = 0, first_page = 0;
    if (threadIdx.x < rows) place_of(p, w, w.first_folded + threadIdx.x, row, head);
    if (warp == 5 && lane < copies) first_page = table[p.paging.page_of(w.begin + lane * rows_per_copy)];
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp < 5) {
        // the queries, a thread a row, while warp 5 already brings the first blocks
        const int r = threadIdx.x;
        if (r < kTcRows) {
            const __nv_bfloat16* src = (const __nv_bfloat16*)p.q + (int64_t)row * p.q_stride + (int64_t)head * dim;
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
                cp_async16(q_tile + (c >> 3) * Tiles::kQSlice + sw128(r, c & 7), c * 8 < dim ? src + c * 8 : src, r < rows && c * 8 < dim);
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_async_smem();
        asm volatile("bar.sync 1, 160;" ::: "memory");            // warps 0..4: the issuer reads the queries after this
    }
    const uint32_t tmem_base = tmem_base_slot;
    const uint32_t tmem_s = tmem_base, tmem_o = tmem_base + kBlock;
    auto tmem_p = [&](int j) { return tmem_o + D + (j & 1) * (kBlock / 2); };
    constexpr uint32_t kStageStep = kBlockBytes >> 4;       // a ring stage further, in the units of a descriptor's address
    int asked_keys = 0, asked_values = 0;                         // blocks that copies were issued for (warp 5)
    int products = 0;                                             // and products (warps 4 and 6)

    if (warp == 5) {
        bool ok = true;
        // block `it` of keys (or values) into its slot, from the pages that the lanes' keys lie in
        auto bring = [&](int it, int page, uint32_t full, uint32_t empty, uint32_t tiles, int which, int& asked) {
            const int s = it % STAGES;
            int go = 1;
            if (lane == 0) {
                go = mbar_wait(empty + 8 * s, ((it / STAGES) & 1) ^ 1, &abort_flag) ? 1 : 0;
                if (go) mbar_expect_tx(full + 8 * s, kBlockBytes);
            }
            go = __shfl_sync(0xffffffffu, go, 0);                 // also orders the announcement before the copies
            if (!go) return false;
            if (lane < copies) {
                const uint32_t dst = tiles + s * kBlockBytes + (uint32_t)(lane * rows_per_copy) * 128;
                const int in_page = p.paging.within(w.begin + it * kBlock + lane * rows_per_copy);
#pragma unroll
                for (int h = 0; h < D / 64; ++h)
                    tma_load_kv(dst + h * kSlice, cache_map, full + 8 * s, h * 64, in_page, w.kv_head, which, page);
            }
            ++asked;
            return true;
        };
        // Keys go one block ahead of values: they are asked for that much earlier,
        // and pages are looked up one block ahead of that.
        auto look_up = [&](int it) {
            return lane < copies && it < n_blocks ? table[p.paging.page_of(w.begin + it * kBlock + lane * rows_per_copy)] : 0;
        };
        int page = first_page, next_page = look_up(1);
        ok = bring(0, page, k_full, k_empty, key_tiles, 0, asked_keys);
        for (int it = 0; it < n_blocks && ok; ++it) {
            const int behind = look_up(it + 2);
            if (it + 1 < n_blocks) ok = bring(it + 1, next_page, k_full, k_empty, key_tiles, 0, asked_keys);
            ok = ok && bring(it, page, v_full, v_empty, value_tiles, 1, asked_values);
            page = next_page;
            next_page = behind;
        }
        if (!ok && lane == 0) {
            abort_flag = 1;
            atomicExch(p.error, 110);
        }
    } else if (warp == 4) {
        if (lane == 0) {
            constexpr uint32_t idesc_qk = idesc_bf16(kTcRows, kBlock, 0);
            // (descriptors are moved by adding to their start-address field, bytes >> 4)
            const uint64_t q_desc = desc_sw128(q_tile, 1), k_desc0 = desc_sw128(key_tiles, 1);
            int s = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (int j = 0; j < n_blocks; ++j) {
                // as soon as the softmax warps hold S_{j-1} in registers the next block's scores may take its place
                if (!mbar_wait(k_full + 8 * s, parity, &abort_flag) || (j > 0 && !mbar_wait(s_free, (j - 1) & 1, &abort_flag))) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t k_desc = k_desc0 + (uint32_t)s * kStageStep;
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma_ss(tmem_s, q_desc + (((kk >> 2) * Tiles::kQSlice + (kk & 3) * 32) >> 4),
                            k_desc + (((kk >> 2) * kSlice + (kk & 3) * 32) >> 4), idesc_qk, kk != 0);
                umma_commit(s_full);
                umma_commit(k_empty + 8 * s);
                ++products;
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
            if (!ok) {
                abort_flag = 1;
                atomicExch(p.error, 120);
            }
        }
    } else if (warp == 6) {
        if (lane == 0) {
            const uint32_t idesc_pv = idesc_bf16(kTcRows, dim, 1);
            const uint64_t v_desc0 = desc_sw128(value_tiles, kSlice >> 4);
            int s = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (int j = 0; j < n_blocks; ++j) {
                if (!mbar_wait(v_full + 8 * s, parity, &abort_flag) || !mbar_wait(p_ready(j), phase(j), &abort_flag)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint64_t v_desc = v_desc0 + (uint32_t)s * kStageStep;
#pragma unroll
                for (int kk = 0; kk < kBlock / 16; ++kk)
                    umma_ts(tmem_o, tmem_p(j) + kk * 8, v_desc + ((kk * 2048) >> 4), idesc_pv, kk != 0 || j != 0);
                umma_commit(o_full(j));
                umma_commit(v_empty + 8 * s);
                ++products;
                if (++s == STAGES) { s = 0; parity ^= 1; }
            }
            if (!ok) {
                abort_flag = 1;
                atomicExch(p.error, 125);
            }
        }
    } else if (warp * 32 < rows) {
        const int r = warp * 32 + lane;                           // row of the tile = lane of tensor memory
        const int64_t slot = slot_of(p, row, head, w.part);
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        // m: the maximum that the stored weights and O are scaled by; it is raised (and O rescaled) only when a block's weights leave
        // their range, which is rare
        float m = kMasked, l = 0.0f;
        bool ok = true;
        // what P_j V_j read and wrote in tensor memory may be touched by this thread again (the fence orders it, the barrier alone does not)
        auto product_done = [&](int j) {
            if (!mbar_wait(o_full(j), phase(j), &abort_flag)) return false;
            tc_fence_after();
            return true;
        };
        const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
        for (int j = 0; j < n_blocks; ++j) {
            if (!mbar_wait(s_full, j & 1, &abort_flag)) { ok = false; break; }
            tc_fence_after();
            uint32_t sc[2][32];
            tmem_load_32(tmem_s + lane_base, sc[0]);
            tmem_load_32(tmem_s + lane_base + 32, sc[1]);
            tmem_wait_ld();
            tc_fence_before();
            mbar_arrive(s_free);                                  // S is in registers: the next block's scores may be computed
            // The weights against the maximum so far, whose block's sum shows whether that is still near enough: a weight above 2^16
            // cannot hide in it, and up to there neither the weights in bfloat16 nor the sums in 32 bits lose anything.  Only
            // otherwise, and in the first block, is the block's maximum looked for and are the weights taken (again) against that.
            uint32_t weights[32];
            float block_sum = 0.0f;
            auto weigh = [&]() {
                const uint64_t neg_m2 = pack2(-m, -m);
                uint64_t ls[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 64; i += 2) {
                    float t0, t1;
                    unpack2(fma2(pack2(__uint_as_float(sc[i >> 5][i & 31]), __uint_as_float(sc[i >> 5][(i & 31) + 1])), scale2, neg_m2), t0, t1);
                    const float p0 = fast_exp2(t0), p1 = fast_exp2(t1);
                    ls[(i >> 1) & 3] = add2(ls[(i >> 1) & 3], pack2(p0, p1));
                    weights[i >> 1] = pack_bf16(p0, p1);
                }
                float lo, hi;
                unpack2(add2(add2(ls[0], ls[1]), add2(ls[2], ls[3])), lo, hi);
                block_sum = lo + hi;
            };
            if (j > 0) weigh();
            if (j == 0 || __any_sync(0xffffffffu, block_sum > 65536.0f)) {
                float mx[4] = {kMasked, kMasked, kMasked, kMasked};
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    mx[(i >> 1) & 1] = max3(mx[(i >> 1) & 1], __uint_as_float(sc[0][i]), __uint_as_float(sc[0][i + 1]));
                    mx[2 + ((i >> 1) & 1)] = max3(mx[2 + ((i >> 1) & 1)], __uint_as_float(sc[1][i]), __uint_as_float(sc[1][i + 1]));
                }
                const float block_max = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale_log2;
                if (j > 0 && !product_done(j - 1)) { ok = false; break; }
                const float m_new = fmaxf(m, block_max), correction = fast_exp2(m - m_new);
                m = m_new;
                l *= correction;
                if (j > 0) {
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        if (c * 16 >= dim) break;
                        uint32_t v[16];
                        asm volatile(
                            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                            : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
                              "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                            : "r"(tmem_o + lane_base + c * 16) : "memory");
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * correction);
                        tmem_store_16(tmem_o + lane_base + c * 16, v);
                    }
                }
                weigh();
            }
            if (j >= 2 && !product_done(j - 2)) { ok = false; break; }               // it has read this buffer
            tmem_store_16(tmem_p(j) + lane_base, weights);
            tmem_store_16(tmem_p(j) + lane_base + 16, weights + 16);
            l += block_sum;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(p_ready(j));
        }
        if (ok && !product_done(n_blocks - 1)) ok = false;
        if (ok) {
            // The row's sums go through shared memory (the queries and the rings are done with: the last product is) and from there
            // as one bulk copy a row: stored from registers, 16 bytes a thread, the tile's 64 KB took 6 us.
            constexpr uint32_t kPitch = D * 4 + 16;               // 16-byte stores of neighbouring rows lie on different banks
            static_assert((size_t)kTcRows * kPitch <= TcShape<D>::kBytes, "the sums fit where the queries and the rings were");
            const uint32_t staged = smem_u32(smem) + r * kPitch;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                if (c * 32 >= dim) break;
                uint32_t v[32];
                tmem_load_32(tmem_o + lane_base + c * 32, v);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                                 ::"r"(staged + (c * 32 + i) * 4), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]) : "memory");
            }
            fence_async_smem();
            if (r < rows) {
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;"
                             ::"l"(p.part_a + slot * dim), "r"(staged), "r"(dim * 4) : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
            if (r < rows) p.part_ml[slot] = make_float2(m, l);
            asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            tc_fence_before();
        } else {
            abort_flag = 1;
            atomicExch(p.error, 130);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        // A wait has run out, perhaps after the warps that issue had left their loops: what is under way is waited for here, where
        // nothing is issued any more, so that no copy or product touches memory that this block has given back.
        if (warp == 5) {
            for (int it = max(0, asked_keys - STAGES); it < asked_keys; ++it) settle(k_full + 8 * (it % STAGES), (it / STAGES) & 1);
            for (int it = max(0, asked_values - STAGES); it < asked_values; ++it) settle(v_full + 8 * (it % STAGES), (it / STAGES) & 1);
        } else if (products > 0) {
            settle((warp == 4 ? k_empty : v_empty) + 8 * ((products - 1) % STAGES), ((products - 1) / STAGES) & 1);
        }
        __syncthreads();
    }
    if (warp == 4) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Tiles::kColumns) : "memory");
    }
}

// Launched behind the kernel of the rows' own keys, whose blocks let it start once they have waited for what was in front of them:
// so everything this kernel reads is there from the start, and its blocks fill the multiprocessors as those end.  What the
// kernel behind reads of both is there once this one is done, so it waits for the one in front before it ends.
template <int D>
__global__ void __launch_bounds__(kTcThreads, kTcBlocks<D>)
shared_tc_kernel(const __grid_constant__ CUtensorMap cache_map, const SharedParams p) {
    extern __shared__ __align__(1024) unsigned char tc_smem[];
    pdl_trigger();
    Work w;
    if (smem_u32(tc_smem) & 1023u) {                              // never expected: refuse rather than compute garbage
        if (threadIdx.x == 0) atomicExch(p.error, 199);
    } else if (find_common<kTcRows>(p, blockIdx.x, w)) {
        attend_tc<D>(p, w, &cache_map, tc_smem);
    }
    if (blockIdx.x == 0) pdl_wait();          // (one block is enough; those without work must not stand in the others' way)
}

// ------------------------------------------------------------------------------------------------ 32-bit

constexpr int kF32Rows = 8;                   // folded rows of a warp
constexpr int kF32Warps = 4;
constexpr int kF32Keys = 32;                  // keys of a tile
constexpr int kF32Aside = 4;                  // keys whose scores a warp sums side by side: with eight rows one a lane
// Columns of a lane.  (8 for 128 too, where two blocks share a multiprocessor instead of three: 64 rows at 2,048 keys 95.0 us instead of
// 96.3, but 8 rows 25.8 instead of 21.2.)
template <int D>
constexpr int kColsF32 = D == 256 ? 8 : 4;

// D: head size padded to 64, 128 or 256.  COLS columns of queries, keys and values are a lane's (one group of four neighbours, or
// two), so keys and values are read whole rows at a time, and one 16-byte load serves 32 multiply-adds; where fewer than 32 lanes
// have a row between them, the parts of a warp take keys of their own.  A lane's products for its keys and the eight rows are
// partial sums, which the lanes exchange in rounds, half as many each, until every lane has one score: as many exchanges for 32 scores
// as lanes share a row, less one.  Rows go in packed pairs.
template <int D, int COLS>
struct RowsF32 {
    static constexpr int kCols = COLS, kLanes = D / COLS, kParts = 32 / kLanes;
    static constexpr int kApart = kLanes * 4;                     // from a lane's first group of columns to its second
    uint64_t query[kF32Rows / 2][kCols], o[kF32Rows / 2][kCols];
    // of row lane % 8: the maximum, and the sum over the keys that this lane weighs
    float m, l;

    // A lane's columns of a row, `from` the first of them, zeros from column `left` on (a multiple of four).
    static __device__ __forceinline__ void load(const float* from, int left, float (&v)[kCols]) {
#pragma unroll
        for (int i = 0; i < kCols / 4; ++i) {
            float4 four = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i * kApart < left) four = *reinterpret_cast<const float4*>(from + i * kApart);
            *reinterpret_cast<float4*>(v + i * 4) = four;
        }
    }

    __device__ __forceinline__ void begin(const SharedParams& p, const Work& w, int first, int rows, int col) {
        m = kMasked;
        l = 0.0f;
#pragma unroll
        for (int pair = 0; pair < kF32Rows / 2; ++pair) {
            float q[2][kCols];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int c = 0; c < kCols; ++c) q[i][c] = 0.0f;
                const int r = (pair * 2 + i) ^ (threadIdx.x & 7);  // (`tile` says why)
                if (r < rows) {
                    int row, head;
                    place_of(p, w, first + r, row, head);
                    load((const float*)p.q + (int64_t)row * p.q_stride + (int64_t)head * p.head_dim + col, p.head_dim - col, q[i]);
                }
            }
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                query[pair][c] = pack2(q[0][c], q[1][c]);
                o[pair][c] = 0;
            }
        }
    }

    // `count` of KEYS keys; key(j) and value(j): this lane's columns of the j-th (those beyond `count` are masked); weights: room for
    // KEYS x 8 numbers of this warp.
    template <int KEYS, typename Key, typename Value>
    __device__ __forceinline__ void tile(float* weights, int count, float scale, Key key, Value value) {
        constexpr int GROUPS = KEYS / kF32Aside, MINE = kF32Aside / kParts;
        static_assert(kF32Rows * MINE == kLanes, "a score a lane");
        const int lane = threadIdx.x & 31, mine = lane / kLanes;
        // Exchanges without a choice: in round r a lane keeps the lower half of its sums and gives the upper away, as lanes whose number
        // has bit r hold their keys (rounds of 8 and more) and query rows (below) with that bit turned over.
        const int turned = (lane >> 3) & (MINE - 1);
        float score[GROUPS];
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            float k[MINE][kCols];
            uint64_t part[kLanes / 2];                            // pairs of rows, key by key
#pragma unroll
            for (int a = 0; a < MINE; ++a) key(g * kF32Aside + mine * MINE + (a ^ turned), k[a]);
#pragma unroll
            for (int a = 0; a < MINE; ++a)
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    const uint64_t twice = pack2(k[a][c], k[a][c]);
#pragma unroll
                    for (int pair = 0; pair < kF32Rows / 2; ++pair) {
                        uint64_t& sum = part[a * (kF32Rows / 2) + pair];
                        sum = c == 0 ? mul2(query[pair][c], twice) : fma2(query[pair][c], twice, sum);
                    }
                }
            float lo, hi;
#pragma unroll
            for (int r = kLanes / 2; r > 1; r >>= 1) {
#pragma unroll
                for (int i = 0; i < r / 2; ++i) {
                    unpack2(part[i + r / 2], lo, hi);
                    part[i] = add2(part[i], pack2(__shfl_xor_sync(0xffffffffu, lo, r), __shfl_xor_sync(0xffffffffu, hi, r)));
                }
            }
            unpack2(part[0], lo, hi);
            score[g] = (lo + __shfl_xor_sync(0xffffffffu, hi, 1)) * scale;           // of key g * 4 + lane / 8 and row lane % 8
        }
        float high = kMasked;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (g * kF32Aside + lane / kF32Rows >= count) score[g] = -INFINITY;      // 2^(that - m) is 0
            high = fmaxf(high, score[g]);
        }
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 8));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, 16));
        const float m_new = fmaxf(m, high);
        if (__any_sync(0xffffffffu, m_new != m)) {
            const float correction = exp2f(m - m_new);
            m = m_new;
            l *= correction;
#pragma unroll
            for (int pair = 0; pair < kF32Rows / 2; ++pair) {
                const uint64_t c_r = pack2(__shfl_sync(0xffffffffu, correction, pair * 2), __shfl_sync(0xffffffffu, correction, pair * 2 + 1));
#pragma unroll
                for (int c = 0; c < kCols; ++c) o[pair][c] = mul2(o[pair][c], c_r);
            }
        }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const float weight = exp2f(score[g] - m);
            l += weight;
            weights[g * 32 + lane] = weight;
        }
        __syncwarp();
#pragma unroll(kCols == 4 ? 8 : 2)
        for (int j = mine; j < count; j += kParts) {
            float v[kCols];
            value(j, v);
            const ulonglong2 w0 = *reinterpret_cast<const ulonglong2*>(weights + j * kF32Rows);
            const ulonglong2 w1 = *reinterpret_cast<const ulonglong2*>(weights + j * kF32Rows + 4);
#pragma unroll
            for (int c = 0; c < kCols; ++c) {
                const uint64_t twice = pack2(v[c], v[c]);
                o[0][c] = fma2(w0.x, twice, o[0][c]);
                o[1][c] = fma2(w0.y, twice, o[1][c]);
                o[2][c] = fma2(w1.x, twice, o[2][c]);
                o[3][c] = fma2(w1.y, twice, o[3][c]);
            }
        }
        __syncwarp();                                             // (what has been read may be written again)
    }

    // The lanes' shares of l together, and the parts' of o.
    __device__ __forceinline__ void end() {
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
        for (int r = kLanes; r < 32; r <<= 1)
#pragma unroll
            for (int pair = 0; pair < kF32Rows / 2; ++pair)
#pragma unroll
                for (int c = 0; c < kCols; ++c) o[pair][c] = add2(o[pair][c], __shfl_xor_sync(0xffffffffu, o[pair][c], r));
    }

    __device__ __forceinline__ void store(int row, float* to, int left) const {      // row: known when this is compiled
#pragma unroll
        for (int c = 0; c < kCols; c += 4) {
            float v[4][2];
#pragma unroll
            for (int i = 0; i < 4; ++i) unpack2(o[row / 2][c + i], v[i][0], v[i][1]);
            if (c / 4 * kApart < left)
                *reinterpret_cast<float4*>(to + c / 4 * kApart) = make_float4(v[0][row & 1], v[1][row & 1], v[2][row & 1], v[3][row & 1]);
        }
    }
};

// A tile of eight folded rows against a run of keys, whose tiles of 32 the four warps take in turns, straight from memory: for few
// rows, where the latency of a load after the look-up before it is what a call waits for (8 beams at 1,111 keys of 32 heads of 64:
// 13 us).  (A lane a key instead, its row read 16 bytes at a time: 131 us for 16 rows at 4,096 keys of 32 heads of 128 where this
// took 67, bound by the cache lines that each load touches.)
template <int D>
__device__ void attend_f32(const SharedParams& p, const Work& w, float* smem) {
    using Rows = RowsF32<D, kColsF32<D>>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int dim = p.head_dim, col = lane % Rows::kLanes * 4;
    float* weights = smem + warp * (kF32Keys * kF32Rows);                            // [key][row] of this warp
    int64_t* places = reinterpret_cast<int64_t*>(smem + kF32Warps * kF32Keys * kF32Rows) + warp * kF32Keys;    // where its keys lie
    Rows rows;
    rows.begin(p, w, w.first_folded, min(kF32Rows, w.folded - w.first_folded), col);
    const int* table = p.table + (int64_t)w.row * p.table_stride;
    const int64_t head_block = (int64_t)p.paging.size * dim;
    const int64_t page_block = 2 * (int64_t)p.kv_heads * head_block;
    const float* keys = (const float*)p.cache + (int64_t)w.kv_head * head_block + col;
    const float* values = keys + (int64_t)p.kv_heads * head_block;
    for (int key0 = w.begin + warp * kF32Keys; key0 < w.end; key0 += kF32Warps * kF32Keys) {
        const int key = min(key0 + lane, w.end - 1);              // (beyond the end: the last key once more, masked)
        places[lane] = (int64_t)table[p.paging.page_of(key)] * page_block + (int64_t)p.paging.within(key) * dim;
        __syncwarp();
        rows.template tile<kF32Keys>(weights, w.end - key0 < kF32Keys ? w.end - key0 : kF32Keys, p.scale_log2,
                                     [&](int j, float (&v)[Rows::kCols]) { Rows::load(keys + places[j], dim - col, v); },
                                     [&](int j, float (&v)[Rows::kCols]) { Rows::load(values + places[j], dim - col, v); });
    }
    rows.end();
    __syncthreads();
    float* ml = smem;
    float* acc = ml + kF32Warps * kF32Rows * 2;
    if (lane < kF32Rows) {
        ml[(warp * kF32Rows + lane) * 2] = rows.m;
        ml[(warp * kF32Rows + lane) * 2 + 1] = rows.l;
    }
    if (lane < Rows::kLanes) {
#pragma unroll
        for (int r = 0; r < kF32Rows; ++r) rows.store(r, acc + (warp * kF32Rows + r) * D + col, D);
    }
    __syncthreads();
    leave_run<float, kF32Rows, D, kF32Warps>(p, w, ml, acc);
}

template <int D>
__global__ void __launch_bounds__(kF32Warps * 32, D <= 128 ? 4 : 2) shared_f32_kernel(const SharedParams p) {
    extern __shared__ __align__(128) float f32_smem[];
    pdl_wait();
    pdl_trigger();
    Work w;
    // (wide: the common parts are the next kernel's)
    if (p.wide ? find_tail<kF32Rows>(p, blockIdx.x, w) : find_work<kF32Rows>(p, blockIdx.x, w)) attend_f32<D>(p, w, f32_smem);
    else if (p.direct) leave_nothing<float, kF32Rows>(p, w);
}

template <int D>
constexpr size_t f32_bytes() {
    constexpr size_t tiles = (size_t)kF32Warps * kF32Keys * (kF32Rows + 2);      // weights, and where the keys lie
    constexpr size_t meet = (size_t)kF32Warps * kF32Rows * (2 + D);
    return (tiles > meet ? tiles : meet) * sizeof(float);
}

// Common parts of groups with more folded rows: four warps with eight rows each against the same keys and values, which go through
// shared memory once for all of them, in asynchronous copies.  32 rows of 32 heads on 8 of 128 at 8,192 keys: 142 us, 4.3 GFLOP,
// 30 TFLOP/s of some 74 that the multiply-adds have (353 us with tiles of eight rows).  Bound by instructions: of 62 for a key and
// eight rows 32 are packed multiply-adds, which take the pipe two cycles each, 12 the exchanges, the rest loads and doubled operands;
// with a choice between two sums in front of each exchange it took 162.
constexpr int kWideRows = kF32Warps * kF32Rows;
template <int D>
constexpr int kWideKeys = D <= 128 ? 32 : 16;
template <int D>
constexpr int kWideStages = D == 64 ? 3 : 2;
template <int D>
constexpr size_t wide_bytes() {
    return ((size_t)kWideStages<D> * 2 * kWideKeys<D> * D + (size_t)kF32Warps * kWideKeys<D> * kF32Rows) * sizeof(float);
}

template <int D>
__device__ void attend_f32_wide(const SharedParams& p, const Work& w, float* smem) {
    using Rows = RowsF32<D, kColsF32<D>>;
    constexpr int KEYS = kWideKeys<D>, STAGES = kWideStages<D>, CH = D / 4, PASSES = KEYS * CH / (kF32Warps * 32);
    constexpr int kTile = KEYS * D;                               // numbers of a tile of keys, or of values
    static_assert(kBlock % KEYS == 0, "a common part ends with a tile: no key is masked");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int dim = p.head_dim, col = lane % Rows::kLanes * 4;
    const int first = w.first_folded + warp * kF32Rows, here = min(kF32Rows, w.folded - first);     // (0 or less: none for this warp)
    float* weights = smem + STAGES * 2 * kTile + warp * (KEYS * kF32Rows);
    const int* table = p.table + (int64_t)w.row * p.table_stride;
    const int64_t head_block = (int64_t)p.paging.size * dim;
    const int64_t page_block = 2 * (int64_t)p.kv_heads * head_block, v_offset = (int64_t)p.kv_heads * head_block;
    const float* base = (const float*)p.cache + (int64_t)w.kv_head * head_block;
    const int tiles = (w.end - w.begin) / KEYS;
    // a lane's key of a tile: its page is looked up one tile ahead of the copies
    auto look_up = [&](int t) { return t < tiles && lane < KEYS ? table[p.paging.page_of(w.begin + t * KEYS + lane)] : 0; };
    auto bring = [&](int t, int page) {
        const int64_t place = (int64_t)page * page_block + (int64_t)p.paging.within(w.begin + t * KEYS + (lane < KEYS ? lane : 0)) * dim;
        const uint32_t dst = smem_u32(smem + (t % STAGES) * 2 * kTile);
#pragma unroll
        for (int pass = 0; pass < PASSES; ++pass) {
            const int idx = pass * (kF32Warps * 32) + (int)threadIdx.x, key = idx / CH, c = idx % CH;
            const float* src = base + __shfl_sync(0xffffffffu, place, key) + c * 4;
            const bool ok = c * 4 < dim;
            cp_async16(dst + idx * 16, ok ? src : base, ok);
            cp_async16(dst + kTile * 4 + idx * 16, ok ? src + v_offset : base, ok);
        }
    };
    int page = look_up(0);
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t) {
        if (t < tiles) bring(t, page);
        cp_async_commit();
        page = look_up(t + 1);
    }
    Rows rows;
    rows.begin(p, w, first, here, col);
    for (int t = 0; t < tiles; ++t) {
        cp_async_wait<STAGES - 2>();
        __syncthreads();                                          // tile t is there, and nobody reads tile t - 1 any more
        if (t + STAGES - 1 < tiles) {
            bring(t + STAGES - 1, page);
            page = look_up(t + STAGES);
        }
        cp_async_commit();
        const float* keys = smem + (t % STAGES) * 2 * kTile + col;
        if (here > 0)
            rows.template tile<KEYS>(weights, KEYS, p.scale_log2, [&](int j, float (&v)[Rows::kCols]) { Rows::load(keys + j * D, D, v); },
                                     [&](int j, float (&v)[Rows::kCols]) { Rows::load(keys + kTile + j * D, D, v); });
    }
    if (here <= 0) return;
    rows.end();
    int64_t slot = 0;
    if (lane < here) {
        int row, head;
        place_of(p, w, first + lane, row, head);
        slot = slot_of(p, row, head, w.part);
        p.part_ml[slot] = make_float2(rows.m, rows.l);
    }
#pragma unroll
    for (int r = 0; r < kF32Rows; ++r) {
        const int64_t to = __shfl_sync(0xffffffffu, slot, r);
        if (r < here && lane < Rows::kLanes) rows.store(r, p.part_a + to * dim + col, dim - col);
    }
}

// (launched as shared_tc_kernel is)
template <int D>
__global__ void __launch_bounds__(kF32Warps * 32, D == 64 ? 4 : D == 128 ? 3 : 2) shared_f32_wide_kernel(const SharedParams p) {
    extern __shared__ __align__(128) float f32_smem[];
    pdl_trigger();
    Work w;
    if (find_common<kWideRows>(p, blockIdx.x, w)) attend_f32_wide<D>(p, w, f32_smem);
    if (blockIdx.x == 0) pdl_wait();
}

// ------------------------------------------------------------------------------------------------ the runs put together

// A warp a (row, head).  Its lanes read the maxima and sums of all runs at once (four a lane: kMaxParts), and their weights stay in
// registers; then LANES lanes read a run's sums, 16 bytes each (for more than 128 columns twice), and 32 / LANES runs side by
// side, eight loads under way a lane.  64 rows of 32 heads of 128 and 19 runs, 20 MB, most of it still in L2: 5 us.  (One load of a
// maximum after the other, a run at a time, took 31.)
constexpr int kMaxParts = 128;
template <typename T, int LANES>
__global__ void __launch_bounds__(128) shared_join_kernel(const SharedParams p) {
    const int lane = threadIdx.x & 31;
    const int64_t index = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (index >= (int64_t)p.rows * p.heads) {
        pdl_wait();
        return;
    }
    const int row = (int)(index / p.heads), head = (int)(index % p.heads);
    // The runs that the row has: the same rule as where they were made.  (The kernel in front lets this one start only once it has
    // itself waited for what made the index arrays, so they may be read before its results are waited for.)
    const int common = common_keys(p, p.common[row]), last = min(p.positions[row] + 1, p.table_keys);
    int of_prefix = 0, of_tail = 0;
    if (common > 0) {
        const int run = run_blocks(common / kBlock, p.prefix_parts, p.prefix_run);
        of_prefix = (common / kBlock + run - 1) / run;
    }
    if (last > common) {
        const int blocks = (last - common + kBlock - 1) / kBlock, run = run_blocks(blocks, p.tail_parts, p.tail_run);
        of_tail = (blocks + run - 1) / run;
    }
    const int64_t slot = slot_of(p, row, head, 0);
    const int parts = of_prefix + of_tail, gap = p.prefix_parts - of_prefix;      // run s is in slot s, or s + gap behind the common part
    float weight[kMaxParts / 32], sum = 0.0f, big = kMasked;
    float2 ml[kMaxParts / 32];
    pdl_wait();
    pdl_trigger();
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) {
        const int s = i * 32 + lane;
        ml[i] = s < parts ? p.part_ml[slot + (s < of_prefix ? s : s + gap)] : make_float2(kMasked, 0.0f);
        big = fmaxf(big, ml[i].x);
    }
    big = warp_max(big);
#pragma unroll
    for (int i = 0; i < kMaxParts / 32; ++i) {
        weight[i] = i * 32 + lane < parts ? exp2f(ml[i].x - big) : 0.0f;
        sum += weight[i] * ml[i].y;
    }
    sum = warp_sum(sum);
    constexpr int AHEAD = 8;                                                      // loads under way
    constexpr int ASIDE = 32 / LANES, TAKES = LANES == 32 ? 2 : 1;                // runs side by side; 16-byte columns of a lane
    const int who = lane / LANES, col = (lane % LANES) * 4;
    float4 a[TAKES];
#pragma unroll
    for (int c = 0; c < TAKES; ++c) a[c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float* from = p.part_a + slot * p.head_dim;
    for (int i = 0; i * 32 < parts; ++i) {
        float chunk = 0.0f;
#pragma unroll
        for (int k = 0; k < kMaxParts / 32; ++k) chunk = k == i ? weight[k] : chunk;
        const int here = min(32, parts - i * 32);
        for (int s0 = 0; s0 < here; s0 += ASIDE * AHEAD) {
            float4 v[AHEAD][TAKES];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int run = i * 32 + min(s0 + u * ASIDE + who, here - 1);     // (beyond the last: the last once more, with no weight)
                const float* of_run = from + (int64_t)(run < of_prefix ? run : run + gap) * p.head_dim;
#pragma unroll
                for (int c = 0; c < TAKES; ++c)
                    v[u][c] = *reinterpret_cast<const float4*>(of_run + min(col + c * 128, p.head_dim - 4));
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int s = s0 + u * ASIDE + who;
                const float w = __shfl_sync(0xffffffffu, chunk, s & 31) * (s < here ? 1.0f : 0.0f);
#pragma unroll
                for (int c = 0; c < TAKES; ++c) {
                    a[c].x = fmaf(w, v[u][c].x, a[c].x);
                    a[c].y = fmaf(w, v[u][c].y, a[c].y);
                    a[c].z = fmaf(w, v[u][c].z, a[c].z);
                    a[c].w = fmaf(w, v[u][c].w, a[c].w);
                }
            }
        }
    }
    const float inverse = parts > 0 ? 1.0f / sum : 0.0f;
    T* out = (T*)p.out + (int64_t)row * p.out_stride + (int64_t)head * p.head_dim;
#pragma unroll
    for (int c = 0; c < TAKES; ++c) {
        float v[4] = {a[c].x, a[c].y, a[c].z, a[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int o = LANES; o < 32; o <<= 1) v[e] += __shfl_xor_sync(0xffffffffu, v[e], o);
            v[e] *= inverse;
        }
        if (who == 0 && col + c * 128 < p.head_dim) {
#pragma unroll
            for (int e = 0; e < 4; ++e) Elem<T>::store(out + col + c * 128 + e, v[e]);
        }
    }
}

// What a kernel is told once a device: the shared memory that it may ask for, and that the multiprocessors be set up for the largest
// (kernels that follow each other without a gap: one that asks for little must not leave the next one little).
int set_up(const void* kernel, size_t smem) {
    static std::mutex lock;
    static std::set<std::pair<const void*, int>> done;
    int device = 0;
    if (const cudaError_t err = cudaGetDevice(&device)) return (int)err;
    std::lock_guard<std::mutex> guard(lock);
    if (done.count({kernel, device})) return 0;
    if (smem > 48 * 1024)
        if (const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return (int)err;
    if (const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared))
        return (int)err;
    try {
        done.insert({kernel, device});
    } catch (const std::bad_alloc&) {         // (asked again next time)
    }
    return 0;
}

template <typename Kernel>
int launch(Kernel kernel, int64_t blocks, int threads, size_t smem, const SharedParams& p, cudaStream_t stream) {
    if (blocks > 0x7fffffff) return TB_ERR_BAD_SIZE;
    if (const int err = set_up((const void*)kernel, smem)) return err;
    if (cudaError_t err = tb_launch_pdl(kernel, dim3((unsigned)blocks), dim3(threads), smem, stream, p)) return (int)err;
    return tb_launch_status();
}

// warps 2: blocks of two warps (where there are enough of them to fill the chip), else as many as share a multiprocessor in pairs.
template <int D, bool ONE>
int launch_mma(int warps, int64_t blocks, const SharedParams& p, cudaStream_t stream) {
    if (warps == 2) return launch(shared_mma_kernel<D, 2, ONE>, blocks, 64, mma_bytes<D, 2>(), p, stream);
    return launch(shared_mma_kernel<D, kWarps<D>, ONE>, blocks, kWarps<D> * 32, mma_bytes<D, kWarps<D>>(), p, stream);
}
template <int D>
int launch_mma(int warps, int64_t blocks, const SharedParams& p, cudaStream_t stream) {
    return p.paging.size % kKeys == 0 ? launch_mma<D, true>(warps, blocks, p, stream) : launch_mma<D, false>(warps, blocks, p, stream);
}

template <int D>
int launch_tc(const CUtensorMap& map, int64_t blocks, const SharedParams& p, cudaStream_t stream) {
    if (blocks > 0x7fffffff) return TB_ERR_BAD_SIZE;
    const size_t smem = TcShape<D>::kBytes;
    if (const int err = set_up((const void*)shared_tc_kernel<D>, smem)) return err;
    if (cudaError_t launched = tb_launch_pdl(shared_tc_kernel<D>, dim3((unsigned)blocks), dim3(kTcThreads), smem, stream, map, p))
        return (int)launched;
    return tb_launch_status();
}

}  // namespace

// Folded rows of a tile: what `tiles` counts.  wide: the form for groups of more folded rows.
TB_EXPORT int tb_attention_shared_tile(int dtype, int wide) {
    return dtype == TB_F32 ? (wide ? kWideRows : kF32Rows) : wide ? kTcRows : kRows;
}

// Whether that form takes these sizes (bfloat16: on the tcgen05 tensor cores).
TB_EXPORT int tb_attention_shared_wide(int dtype, int head_dim, int page_size) {
    if (dtype == TB_F32) return 1;
    return dtype == TB_BF16 && head_dim <= 256 && page_size >= 8 && (page_size & (page_size - 1)) == 0;
}

// rows of q and out: [rows, heads * head_dim] with a stride; positions[b]: the last key of row b (-1: none); table: [rows, columns]
// pages; members, group_start, leader, prefix, common: the groups (SharedParams); tiles: the tiles of all groups with keys in common,
// ceil(rows of the group * heads / kv_heads / tile) each, no fewer.  prefix[g] is at most positions[b] + 1 for the rows of the group.
// part_a, part_ml: rows * heads * (prefix_parts + tail_parts) * (head_dim and 2) floats; none where nothing is in common and every
// row is one run.
// The arguments come as one run of bytes (as declared here, nothing between them): a call of so many cost the host 3 us more.
struct SharedCall {
    const void* q;
    int64_t q_stride;
    void* out;
    int64_t out_stride;
    const void* cache;
    const int *positions, *table, *members, *group_start, *leader, *prefix, *common;
    float *part_a, *part_ml;
    int64_t part_floats;
    int* error;
    int table_stride, table_columns, rows, groups, heads, kv_heads, head_dim, page_size;
    int tiles, prefix_parts, prefix_run, tail_parts, tail_run, warps, wide, cache_pages, dtype;
    float scale;
};
static_assert(sizeof(SharedCall) == 16 * 8 + 18 * 4, "nothing between the arguments");

TB_EXPORT int tb_attention_shared(const void* packed, cudaStream_t stream) {
    SharedCall call;
    memcpy(&call, packed, sizeof(call));
    const int rows = call.rows, groups = call.groups, heads = call.heads, kv_heads = call.kv_heads, head_dim = call.head_dim;
    const int page_size = call.page_size, tiles = call.tiles, prefix_parts = call.prefix_parts, tail_parts = call.tail_parts;
    const int warps = call.warps, wide = call.wide, dtype = call.dtype;
    if (rows == 0) return 0;
    if (dtype != TB_F32 && dtype != TB_BF16) return TB_ERR_BAD_DTYPE;
    if (rows < 0 || groups < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads != 0 || page_size < 1 || tiles < 0) return TB_ERR_BAD_SIZE;
    if (head_dim < 16 || head_dim > 256 || head_dim % 16 != 0) return TB_ERR_BAD_SIZE;
    if (prefix_parts < 0 || tail_parts < 1 || prefix_parts + tail_parts > kMaxParts || call.prefix_run < 1 || call.tail_run < 1) return TB_ERR_BAD_SIZE;
    const int element = dtype == TB_F32 ? 4 : 2;
    if (((uintptr_t)call.q | (uintptr_t)call.out | (uintptr_t)call.cache | (uintptr_t)call.part_a) % 16 != 0) return TB_ERR_BAD_ALIGN;
    if ((call.q_stride * element) % 16 != 0) return TB_ERR_BAD_ALIGN;
    const int64_t parts = prefix_parts == 0 && tail_parts == 1 ? 0 : (int64_t)rows * heads * (prefix_parts + tail_parts);
    if (parts > 0 && (call.part_a == nullptr || call.part_ml == nullptr || call.part_floats < parts * head_dim)) return -5;
    if (wide && (!tb_attention_shared_wide(dtype, head_dim, page_size) || call.error == nullptr)) return TB_ERR_BAD_SIZE;
    SharedParams p;
    p.q = call.q;
    p.out = call.out;
    p.cache = call.cache;
    p.positions = call.positions;
    p.table = call.table;
    p.members = call.members;
    p.group_start = call.group_start;
    p.leader = call.leader;
    p.prefix = call.prefix;
    p.common = call.common;
    p.part_a = call.part_a;
    p.part_ml = (float2*)call.part_ml;
    p.q_stride = call.q_stride;
    p.out_stride = call.out_stride;
    p.table_stride = call.table_stride;
    const int64_t keys = (int64_t)call.table_columns * page_size;
    p.table_keys = (int)(keys < 0x7fffff00 ? keys : 0x7fffff00);
    p.rows = rows;
    p.groups = groups;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.fold = heads / kv_heads;
    p.head_dim = head_dim;
    p.tiles = tiles;
    p.prefix_parts = prefix_parts;
    p.prefix_run = call.prefix_run;
    p.tail_parts = tail_parts;
    p.tail_run = call.tail_run;
    p.paging = tb_paging(page_size);
    p.scale_log2 = call.scale * kLog2e;
    p.wide = wide;
    p.direct = prefix_parts == 0 && tail_parts == 1;
    p.error = call.error;
    const int tile = dtype == TB_F32 ? kF32Rows : kRows;                 // of the parts behind
    const int64_t of_common = (int64_t)tiles * kv_heads * prefix_parts;
    const int64_t blocks = (wide ? 0 : of_common) + (int64_t)rows * ((p.fold + tile - 1) / tile) * kv_heads * tail_parts;
    int status;
    if (dtype == TB_F32) {
        if (head_dim <= 64) status = launch(shared_f32_kernel<64>, blocks, kF32Warps * 32, f32_bytes<64>(), p, stream);
        else if (head_dim <= 128) status = launch(shared_f32_kernel<128>, blocks, kF32Warps * 32, f32_bytes<128>(), p, stream);
        else status = launch(shared_f32_kernel<256>, blocks, kF32Warps * 32, f32_bytes<256>(), p, stream);
        if (status == 0 && wide && of_common > 0) {
            if (head_dim <= 64) status = launch(shared_f32_wide_kernel<64>, of_common, kF32Warps * 32, wide_bytes<64>(), p, stream);
            else if (head_dim <= 128) status = launch(shared_f32_wide_kernel<128>, of_common, kF32Warps * 32, wide_bytes<128>(), p, stream);
            else status = launch(shared_f32_wide_kernel<256>, of_common, kF32Warps * 32, wide_bytes<256>(), p, stream);
        }
    } else {
        if (head_dim <= 32) status = launch_mma<32>(warps, blocks, p, stream);
        else if (head_dim <= 64) status = launch_mma<64>(warps, blocks, p, stream);
        else if (head_dim <= 128) status = launch_mma<128>(warps, blocks, p, stream);
        else status = launch_mma<256>(warps, blocks, p, stream);
        if (status == 0 && wide && of_common > 0) {
            CUtensorMap map;
            if (!make_cache_map(&map, call.cache, call.cache_pages, kv_heads, page_size, kBlock, head_dim)) return TB_ERR_BAD_SIZE;
            status = head_dim <= 64 ? launch_tc<64>(map, of_common, p, stream)
                     : head_dim <= 128 ? launch_tc<128>(map, of_common, p, stream) : launch_tc<256>(map, of_common, p, stream);
        }
    }
    if (status != 0 || p.direct) return status;
    const int64_t joins = ((int64_t)rows * heads + 3) / 4;
    if (dtype == TB_F32)
        return launch(head_dim <= 32 ? shared_join_kernel<float, 8> : head_dim <= 64 ? shared_join_kernel<float, 16>
                                                                                     : shared_join_kernel<float, 32>,
                      joins, 128, 0, p, stream);
    return launch(head_dim <= 32 ? shared_join_kernel<__nv_bfloat16, 8> : head_dim <= 64 ? shared_join_kernel<__nv_bfloat16, 16>
                                                                                         : shared_join_kernel<__nv_bfloat16, 32>,
                  joins, 128, 0, p, stream);
}
