// Pages (or state slots) of several stores copied within each store, in one launch.
//
//   store[e][target_i] = store[e][source_i]     for every entry e of the store and every move i
//
// A store is [entries][pages][page bytes] of any element type.  No target is named twice and none is a source, so the
// order of the moves cannot matter; the host entry refuses a call in which that does not hold, or whose pages lie
// outside their store, before anything is launched.
//
// The moves travel in the launch's own parameters (a constant bank, read by every block at the same index), so a fork
// needs no copy of an index array to the device, no buffer that has to outlive the call, and no wait.  Calls of more
// moves than fit the parameters of one launch are cut into several launches.
//
// Bound by HBM: every byte is read once and written once.  A block copies one piece of one page with 16-byte loads, all
// of a thread's loads in flight before its first store.  1,500 pages of a 32-bit cache moved down, 1.57 GB read and written: 244 us,
// the measured copy rate (6.4 TB/s); states and last pages of 31 forks, 2.21 GB: 334 us, 6.6 TB/s.  A fork of a few pages is bound
// by the host: 7.5 us a call, of which the launch is 2.
#include <new>
#include <vector>

#include "common.cuh"

namespace {

constexpr int kThreads = 128;
constexpr int kMaxStores = 8;      // stores of one launch
constexpr int kFewMoves = 48;      // moves of the small form (a launch copies its parameters: 2 us of host time for the large one)
constexpr int kManyMoves = 3968;   // of the large one: 31,744 of the 32,764 bytes that a launch's parameters may have

struct Store {
    char* base;
    int64_t pitch, size;           // bytes from an entry to the next, of a page
    int64_t first_piece;           // pieces of the stores in front
    int first_move, moves, pieces; // its moves in the list; pieces of a page
    int width;                     // bytes of a load: 16, 4 or 1
};

template <int MOVES>
struct Params {
    Store stores[kMaxStores];
    int2 moves[MOVES];             // source, target
    int count;
    int piece;                     // bytes of a piece
};

template <typename T, int UNROLL>
__device__ __forceinline__ void copy_piece(const char* from, char* to, int bytes) {
    const T* in = reinterpret_cast<const T*>(from);
    T* out = reinterpret_cast<T*>(to);
    const int count = bytes / (int)sizeof(T);
    for (int i0 = 0; i0 < count; i0 += UNROLL * kThreads) {
        T held[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = i0 + u * kThreads + (int)threadIdx.x;
            if (i < count) held[u] = in[i];
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = i0 + u * kThreads + (int)threadIdx.x;
            if (i < count) out[i] = held[u];
        }
    }
}

template <int MOVES>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ Params<MOVES> p) {
    const int64_t piece = blockIdx.x;
    int s = 0;
    while (s + 1 < p.count && piece >= p.stores[s + 1].first_piece) ++s;
    const Store& store = p.stores[s];
    const int64_t at = piece - store.first_piece;
    const int part = (int)(at % store.pieces);
    const int64_t which = at / store.pieces;
    const int2 move = p.moves[store.first_move + (int)(which % store.moves)];
    char* entry = store.base + (which / store.moves) * store.pitch;
    const int64_t offset = (int64_t)part * p.piece;
    const int bytes = (int)min((int64_t)p.piece, store.size - offset);
    const char* from = entry + (int64_t)move.x * store.size + offset;
    char* to = entry + (int64_t)move.y * store.size + offset;
    if (store.width == 16) copy_piece<uint4, 8>(from, to, bytes);
    else if (store.width == 4) copy_piece<uint32_t, 8>(from, to, bytes);
    else copy_piece<uint8_t, 4>(from, to, bytes);
}

template <int MOVES>
int launch(const Params<MOVES>& p, int64_t pieces, cudaStream_t stream) {
    if (pieces > 0x7fffffff) return TB_ERR_BAD_SIZE;
    copy_pages_kernel<MOVES><<<(unsigned)pieces, kThreads, 0, stream>>>(p);
    return tb_launch_status();
}

int piece_bytes(int64_t total) { return total >= (int64_t)(32 << 20) ? 16384 : 4096; }

}  // namespace

constexpr int kErrBadPage = -6, kErrClash = -7, kErrMemory = -8;

// packed: for every store its address, entries, pages, bytes of a page and moves; then, as 32-bit numbers, every store's sources and
// targets.  Returns (launches << 16) + status.
TB_EXPORT int tb_copy_pages(int num_stores, const int64_t* packed, cudaStream_t stream) {
    auto base = [&](int s) { return (char*)packed[s * 5]; };
    auto entries = [&](int s) { return packed[s * 5 + 1]; };
    auto pages = [&](int s) { return packed[s * 5 + 2]; };
    auto size = [&](int s) { return packed[s * 5 + 3]; };
    auto counts = [&](int s) { return (int)packed[s * 5 + 4]; };
    int at_store = 0;
    const int* indices = (const int*)(packed + 5 * (int64_t)num_stores);
    // (asked in the order of the stores, twice)
    auto sources = [&](int s) {
        if (s < at_store) {
            at_store = 0;
            indices = (const int*)(packed + 5 * (int64_t)num_stores);
        }
        for (; at_store < s; ++at_store) indices += 2 * (int64_t)counts(at_store);
        return indices;
    };
    auto targets = [&](int s) { return sources(s) + counts(s); };
    int launches = 0;
    std::vector<uint8_t> seen;
    int64_t total_bytes = 0;
    for (int s = 0; s < num_stores; ++s) {
        if (entries(s) < 0 || pages(s) < 0 || pages(s) > 0x7fffffff || size(s) < 0 || packed[s * 5 + 4] < 0 || packed[s * 5 + 4] > 0x3fffffff)
            return TB_ERR_BAD_SIZE;
        const int n = counts(s);
        const int *source = sources(s), *target = targets(s);
        try {
            seen.assign((size_t)pages(s), 0);
        } catch (const std::bad_alloc&) {
            return kErrMemory;
        }
        for (int i = 0; i < n; ++i) {
            if (source[i] < 0 || source[i] >= pages(s) || target[i] < 0 || target[i] >= pages(s)) return kErrBadPage;
            seen[(size_t)source[i]] = 1;
        }
        for (int i = 0; i < n; ++i) {
            uint8_t& mark = seen[(size_t)target[i]];
            if (mark) return kErrClash;
            mark = 2;
        }
        total_bytes += size(s) * counts(s) * entries(s);
    }
    if (total_bytes == 0) return 0;
    // one launch takes up to kMaxStores stores and as many moves as its parameters hold; a store's moves may go on in the next
    int s = 0, done = 0;
    int64_t moves_left = 0;
    for (int k = 0; k < num_stores; ++k) moves_left += counts(k);
    Params<kFewMoves> few;
    static thread_local Params<kManyMoves> many;       // (32 KB: too large to lay on a caller's stack unasked)
    while (s < num_stores) {
        const bool small = moves_left <= kFewMoves;
        Store* stores = small ? few.stores : many.stores;
        int2* moves = small ? few.moves : many.moves;
        const int room = small ? kFewMoves : kManyMoves;
        const int piece = piece_bytes(total_bytes);
        int used = 0, taken = 0;
        int64_t pieces = 0;
        while (s < num_stores && used < kMaxStores && taken < room) {
            const int n = counts(s) - done < room - taken ? counts(s) - done : room - taken;
            if (n > 0 && entries(s) > 0 && size(s) > 0) {
                Store& store = stores[used++];
                store.base = base(s);
                store.pitch = size(s) * pages(s);
                store.size = size(s);
                const uint64_t all = (uint64_t)(uintptr_t)base(s) | (uint64_t)size(s);
                store.width = all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 1;
                store.first_move = taken;
                store.moves = n;
                store.pieces = (int)((size(s) + piece - 1) / piece);
                store.first_piece = pieces;
                pieces += (int64_t)store.pieces * n * entries(s);
                const int *source = sources(s) + done, *target = targets(s) + done;
                for (int i = 0; i < n; ++i) moves[taken + i] = make_int2(source[i], target[i]);
                taken += n;
            }
            done += n;
            moves_left -= n;
            if (done < counts(s)) break;
            done = 0;
            ++s;
        }
        if (pieces == 0) continue;
        (small ? few.count : many.count) = used;
        (small ? few.piece : many.piece) = piece;
        const int status = small ? launch(few, pieces, stream) : launch(many, pieces, stream);
        if (status != 0) return (launches << 16) + status;
        ++launches;
    }
    return launches << 16;
}
