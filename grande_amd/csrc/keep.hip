// Rows of a paged K/V cache that stay: moving them where they are to lie
// (keep), and choosing them by the weight they have gathered (evict).
#include <algorithm>
#include <string>

#include "choose.h"
#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

namespace {

typedef uint32_t chunk_t __attribute__((ext_vector_type(4)));  // 16 bytes of a row

struct KeepArgs {
    PagedKv kv;
    PagedBatch b;
    KeepRows x;
    int page_shift;
    int64_t waves;  // in all
    int slices;     // in place: a row's slices, a wave each
    int groups;     // apart: waves of a list
};

// The element offset of a cache row of KV head g (below zero: not in the pool).
__device__ inline int64_t row_at(const KeepArgs& a, const int32_t* table, int64_t pages, int64_t row, int64_t g) {
    const int64_t i = row >> a.page_shift;
    if (row < 0 || i >= pages) return -1;
    const int64_t p = table[i];
    if (p < 0 || p >= a.kv.npages) return -1;
    return p * a.kv.page_stride + (g * a.kv.page + (row & (a.kv.page - 1))) * a.kv.head_dim;
}

// Rows j0, j0 + W, .. (U of them, below `end`) of sequence s and KV head g, from
// its rows row(j) to its rows first + j on other pages: 8 head dims at c of each.
template <int U, typename F>
__device__ inline void move_apart(const KeepArgs& a, int64_t s, int64_t g, int64_t first, int64_t j0, int64_t end, int W, int c, F row) {
    int64_t from[U], to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t j = j0 + u * W;
        from[u] = to[u] = -1;
        if (j >= end) continue;
        from[u] = row_at(a, a.b.table + s * a.b.table_ld, a.b.max_pages, row(j), g);
        to[u] = row_at(a, a.x.to_table + s * a.x.to_ld, a.x.to_ld, first + j, g);
    }
    chunk_t k[U], v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (from[u] < 0 || to[u] < 0) continue;
        k[u] = *reinterpret_cast<const chunk_t*>(static_cast<const uint16_t*>(a.kv.k) + from[u] + c);
        v[u] = *reinterpret_cast<const chunk_t*>(static_cast<const uint16_t*>(a.kv.v) + from[u] + c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (from[u] < 0 || to[u] < 0) continue;
        *reinterpret_cast<chunk_t*>(static_cast<uint16_t*>(a.kv.k) + to[u] + c) = k[u];
        *reinterpret_cast<chunk_t*>(static_cast<uint16_t*>(a.kv.v) + to[u] + c) = v[u];
    }
}

// To other pages: no row is read and written, so every wave moves rows of its
// own, U pieces of 1 KiB (512 / D rows each) of K and of V at once.  Bound by the
// bytes: 64 x 8 lists of 1,000 rows of 128 105 us, 5.0 TB/s, what a large copy
// reaches; 4,095 rows each 455 us, 4.7 TB/s.  (U = 2: with 1 too few loads are under
// way, with 4 fewer waves fit a CU, 124 us, with 8 217; non-temporal 106.)
template <int D, int U>
__global__ __launch_bounds__(256) void keep_apart_kernel(KeepArgs a) {
    constexpr int L = D / 8, W = WAVE / L;  // lanes of a row, rows of a piece
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t id = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    if (id >= a.waves) return;
    const int64_t list = id / a.groups, s = list / a.kv.kv_heads, g = list - s * a.kv.kv_heads;
    const int32_t* rows = a.x.rows + (a.x.per_head ? list : s) * a.x.rows_ld;
    move_apart<U>(a, s, g, a.x.first ? a.x.first[s] : 0, (id - list * a.groups) * (U * W) + lane / L, a.x.count, W, lane % L * 8,
                  [&](int64_t j) { return rows[j]; });
}

// In place: an entry that moves has rows[j] >= first + j, so the place that an
// entry writes is read by entries up to its own alone.  One wave takes
// a list's K or V (or a slice of SB bytes of each row) from the first entry on,
// in steps of U pieces, and a wave's loads return in order: an entry has its
// row, and all entries before it theirs, when its place is written.  Loads run
// ahead of the stores: while a step's rows arrive the next step's pages and the
// entries of the one after are asked for.  Bound by a wave's own chain of steps
// where lists are few (one list of 4,000 rows of 256, 16 slices: 82 us), by the
// bytes where they are many (64 x 8 lists of 1,000 rows of 128: 125 us, 4.2 TB/s;
// 12 accepted paths of a few rows: 4.8 us, a launch).
template <int SB>
__global__ __launch_bounds__(256) void keep_in_place_kernel(KeepArgs a) {
    constexpr int L = SB / 16, W = WAVE / L, U = 8;
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t id = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    if (id >= a.waves) return;
    const int slice = int(id % a.slices);
    const int64_t half = id / a.slices, list = half / 2, s = list / a.kv.kv_heads, g = list - s * a.kv.kv_heads;
    uint16_t* x = static_cast<uint16_t*>(half % 2 ? a.kv.v : a.kv.k) + slice * (SB / 2) + lane % L * 8;
    const int32_t *rows = a.x.rows + (a.x.per_head ? list : s) * a.x.rows_ld, *table = a.b.table + s * a.b.table_ld;
    const int64_t first = (a.x.first ? a.x.first[s] : 0) + int64_t(lane / L), count = a.x.count - lane / L;
    const int mask = a.kv.page - 1;
    struct Step {
        int row[U], from[U], to[U];  // source rows, pages of the sources and places (below zero: nothing moves)
    };
    auto entries = [&](int64_t j0, Step& t) {
#pragma unroll
        for (int u = 0; u < U; ++u) t.row[u] = -1;
        if (j0 >= a.x.count) return;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (j0 + u * W < count) t.row[u] = rows[lane / L + j0 + u * W];
    };
    auto pages = [&](int64_t j0, Step& t) {
#pragma unroll
        for (int u = 0; u < U; ++u) t.from[u] = t.to[u] = -1;
        if (j0 >= a.x.count) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = t.row[u], d = first + j0 + u * W;
            const bool moves = r > d && d >= 0 && r >> a.page_shift < a.b.max_pages;
            if (moves) t.from[u] = table[r >> a.page_shift], t.to[u] = table[d >> a.page_shift];
        }
    };
    auto place = [&](int p, int64_t row) {
        return x + p * a.kv.page_stride + (g * a.kv.page + (row & mask)) * a.kv.head_dim;
    };
    auto moves = [&](const Step& t, int u) { return uint64_t(t.from[u]) < uint64_t(a.kv.npages) && uint64_t(t.to[u]) < uint64_t(a.kv.npages); };
    auto load = [&](const Step& t, chunk_t* v) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (moves(t, u)) v[u] = *reinterpret_cast<const chunk_t*>(place(t.from[u], t.row[u]));
    };
    Step now, next, then;
    chunk_t v[U], w[U];
    entries(0, now);
    entries(U * W, next);
    pages(0, now);
    entries(2 * U * W, then);
    pages(U * W, next);
    load(now, v);
    for (int64_t j0 = 0; j0 < a.x.count; j0 += U * W) {
        load(next, w);
        pages(j0 + 2 * U * W, then);
        Step more;
        entries(j0 + 3 * U * W, more);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (moves(now, u)) *reinterpret_cast<chunk_t*>(place(now.to[u], first + j0 + u * W)) = v[u];
        asm volatile("" ::: "memory");
        now = next, next = then, then = more;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = w[u];
    }
}

template <int D>
void launch_apart(hipStream_t s, KeepArgs a) {
    constexpr int W = 512 / D, U = 2;
    a.groups = int((a.x.count + U * W - 1) / (U * W));
    a.waves = a.b.nseq * a.kv.kv_heads * a.groups;
    const int64_t blocks = (a.waves + 3) / 4;
    if (blocks >= MAX_BLOCKS) fail(E_CAPACITY, "kv_keep: too many rows for one call");
    keep_apart_kernel<D, U><<<dim3(unsigned(blocks)), dim3(256), 0, s>>>(a);
}

template <int SB>
void launch_in_place(hipStream_t s, KeepArgs a) {
    a.slices = a.kv.head_dim * 2 / SB;
    a.waves = a.b.nseq * a.kv.kv_heads * 2 * a.slices;
    const int64_t blocks = (a.waves + 3) / 4;
    if (blocks >= MAX_BLOCKS) fail(E_CAPACITY, "kv_keep: too many lists for one call");
    keep_in_place_kernel<SB><<<dim3(unsigned(blocks)), dim3(256), 0, s>>>(a);
}

void move_rows(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const KeepRows& x) {
    KeepArgs a{kv, b, x, log2_of(kv.page), 0, 1, 1};
    if (x.to_table) {
        switch (kv.head_dim) {
            case 64: launch_apart<64>(s, a); break;
            case 128: launch_apart<128>(s, a); break;
            case 256: launch_apart<256>(s, a); break;
            default: launch_apart<512>(s, a);
        }
    } else {
        // Few lists: rows in slices, down to half a cache line each.
        int sb = kv.head_dim * 2;
        while (sb > 64 && b.nseq * kv.kv_heads * 2 * (kv.head_dim * 2 / sb) < 1024) sb /= 2;
        switch (sb) {
            case 64: launch_in_place<64>(s, a); break;
            case 128: launch_in_place<128>(s, a); break;
            case 256: launch_in_place<256>(s, a); break;
            case 512: launch_in_place<512>(s, a); break;
            default: launch_in_place<1024>(s, a);
        }
    }
    OMG_HIP(hipGetLastError());
}

void check_sequences(const PagedBatch& b, const PagedKv& kv, const char* who) {
    PagedBatch own = b;  // (what the tokens and the prefix are does not matter here)
    own.prefix_len = 0;
    check_batch(own, kv, who);
}

// ------------------------------------------------------------------- evict
//
// A workgroup chooses a list's rows: the `recent` last ones and, of those
// before them, the keep - recent of the largest weights (choose.h).  Bound by the
// choice's chain of barriers: 12 lists of 2,300 weights 9 us; 512 lists of 6,100
// 28 us (their 12.5 MB alone 2.5 us).  (512 threads where they hold the list: its
// barriers are shorter, 1,024 take 1.4 us more; past that 1,024, and past these
// the list is read in every pass: 8,000 values by 512 threads 6 us more.)
//
// MOVE: each of a list's `groups` workgroups makes the same choice, which costs
// nothing where they fill places that would be empty, and moves the rows of its
// slice of the places to other pages; the first writes the lists.  (12 lists of
// 2,300 cut to 1,024 rows of 256 12 us, in two launches 15.3; 32 of 4,000 cut to
// 2,000 rows of 128 21 and 22; at 64 the same, at 128 74 and 68, since so few waves
// move rows at less than the rate of a launch of their own.)

constexpr int EVICT_MOVES = 32;  // lists

struct EvictArgs {
    KeepArgs move;  // (with its pool, batch and places)
    EvictRows x;
    int64_t max_len;
    int groups, per;  // MOVE: of a list, and the rows of each
};

template <int T, bool HELD, bool MOVE>
__global__ __launch_bounds__(T) void evict_kernel(EvictArgs a) {
    typedef Choose<T, HELD> C;
    __shared__ typename C::Shared shared;
    extern __shared__ int32_t slice[];  // the rows that the workgroup moves
    const int tid = int(threadIdx.x);
    const int64_t list = MOVE ? blockIdx.x / a.groups : blockIdx.x, s = list / a.move.kv.kv_heads;
    const float* w = a.x.weights + list * a.x.ldw;
    float* kept = a.x.kept + list * a.x.kept_ld;
    int32_t* rows = a.x.rows + list * a.x.keep;
    const int len = a.move.b.lens[s], n = len < 0 ? 0 : len < a.max_len ? len : int(a.max_len);
    const int keep = int(a.x.keep), recent = int(a.x.recent);
    const int part = MOVE ? int(blockIdx.x % a.groups) : 0, from = part * a.per, to = from + a.per < keep ? from + a.per : keep;
    auto place = [&](int rank, int row) {
        if (part == 0) rows[rank] = row;
        if (MOVE && rank >= from && rank < to) slice[rank - from] = row;
    };
    if (n <= keep) {
        for (int i = tid; i < keep; i += T) {
            place(i, i < n ? i : -1);
            if (part == 0 && i < n && kept != w) kept[i] = w[i];
        }
    } else {
        const int old = n - recent, chosen = keep - recent;
        C::run(shared, w, old, uint32_t(chosen), [&](int rank, int row, float x) {
            place(rank, row);
            if (part == 0) kept[rank] = x;
        });
        // The recent rows, and zeros for the rows to come.
        for (int i0 = 0; i0 < recent; i0 += T) {
            const int i = i0 + tid;
            const float x = i < recent ? w[old + i] : 0.0f;
            if (!MOVE) __syncthreads();
            if (i < recent) place(chosen + i, old + i);
            if (i < recent && part == 0) kept[chosen + i] = x;
        }
        __syncthreads();
        if (part == 0)
            for (int i = keep + tid; i < n && i < a.x.kept_ld; i += T) kept[i] = 0.0f;
    }
    if constexpr (MOVE) {
        __syncthreads();
        constexpr int U = 2;
        const int L = a.move.kv.head_dim / 8, W = T / L;
        for (int64_t j = from + tid / L; j < to; j += U * W)
            move_apart<U>(a.move, s, list - s * a.move.kv.kv_heads, 0, j, to, W, tid % L * 8, [&](int64_t j) { return slice[j - from]; });
    }
}

template <int T, bool HELD>
void launch_evict(hipStream_t s, EvictArgs a) {
    const int64_t lists = a.move.b.nseq * a.move.kv.kv_heads;
    // Few lists whose weights are not written over go to other pages in one launch.
    if constexpr (HELD) {
        if (a.x.to_table && a.x.kept != a.x.weights && lists <= EVICT_MOVES) {
            a.groups = int(256 / lists);
            a.per = int((a.x.keep + a.groups - 1) / a.groups);
            a.groups = int((a.x.keep + a.per - 1) / a.per);
            evict_kernel<T, true, true><<<dim3(unsigned(lists * a.groups)), dim3(T), unsigned(a.per) * 4, s>>>(a);
            OMG_HIP(hipGetLastError());
            return;
        }
    }
    if (lists >= MAX_BLOCKS / (T / 256)) fail(E_CAPACITY, "kv_evict: too many lists for one call");
    evict_kernel<T, HELD, false><<<dim3(unsigned(lists)), dim3(T), 0, s>>>(a);
    OMG_HIP(hipGetLastError());
    move_rows(s, a.move.kv, a.move.b, a.move.x);
}

}  // namespace

void launch_kv_keep(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const KeepRows& x) {
    check_kv(kv, "kv_keep");
    check_sequences(b, kv, "kv_keep");
    if (!x.rows) fail(E_INVALID, "kv_keep: null rows");
    if (x.count <= 0 || x.count > b.max_pages * kv.page || x.rows_ld < x.count)
        fail(E_INVALID, "kv_keep: count must be 1 to a sequence's rows and rows_ld hold it");
    if (x.to_table && (x.to_ld <= 0 || x.to_ld > 0x3fffffff / kv.page))
        fail(E_INVALID, "kv_keep: to_ld out of range");
    move_rows(s, kv, b, x);
}

void launch_kv_evict(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const EvictRows& x) {
    check_kv(kv, "kv_evict");
    check_sequences(b, kv, "kv_evict");
    const int64_t max_len = b.max_pages * kv.page;
    if (!x.weights || !x.rows) fail(E_INVALID, "kv_evict: null weights or rows");
    if (x.keep <= 0 || x.recent < 0 || x.recent > x.keep)
        fail(E_INVALID, "kv_evict: keep must be positive and recent 0 to keep");
    if (x.keep > max_len) fail(E_INVALID, "kv_evict: keep must be at most a sequence's rows");
    if (x.ldw < max_len) fail(E_INVALID, "kv_evict: ldw must hold a sequence's rows");
    if (x.kept && x.kept != x.weights && x.kept_ld < x.keep) fail(E_INVALID, "kv_evict: kept_ld must hold keep weights");
    if (x.kept == x.weights && x.kept_ld != x.ldw) fail(E_INVALID, "kv_evict: kept_ld must be ldw in place");
    if (x.to_table && (x.to_ld <= 0 || x.to_ld > 0x3fffffff / kv.page))
        fail(E_INVALID, "kv_evict: to_ld out of range");
    const KeepRows moves{x.rows, x.keep, x.keep, nullptr, 1, x.to_table, x.to_ld};
    const EvictArgs a{KeepArgs{kv, b, moves, log2_of(kv.page), 0, 1, 1}, x, max_len, 1, int(x.keep)};
    if (max_len <= CHOOSE_R * 512)
        launch_evict<512, true>(s, a);
    else if (max_len <= CHOOSE_R * 1024)
        launch_evict<1024, true>(s, a);
    else
        launch_evict<1024, false>(s, a);
}

}  // namespace omg
