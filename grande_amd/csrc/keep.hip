// Rows of a paged K/V cache that stay: moving them where they are to lie
// (keep), and choosing them by the weight they have gathered (evict).
#include <algorithm>
#include <string>

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

// To other pages: no row is read and written, so every wave moves rows of its
// own, U pieces of 1 KiB (512 / D rows each) of K and of V at once.
template <int D, int U>
__global__ __launch_bounds__(256) void keep_apart_kernel(KeepArgs a) {
    constexpr int L = D / 8, W = WAVE / L;  // lanes of a row, rows of a piece
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t id = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    if (id >= a.waves) return;
    const int64_t list = id / a.groups, s = list / a.kv.kv_heads, g = list - s * a.kv.kv_heads;
    const int64_t j0 = (id - list * a.groups) * (U * W) + lane / L;
    const int32_t* rows = a.x.rows + (a.x.per_head ? list : s) * a.x.rows_ld;
    const int64_t first = a.x.first ? a.x.first[s] : 0;
    const int c = lane % L * 8;
    int64_t from[U], to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t j = j0 + u * W;
        from[u] = to[u] = -1;
        if (j >= a.x.count) continue;
        from[u] = row_at(a, a.b.table + s * a.b.table_ld, a.b.max_pages, rows[j], g);
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

// In place: entry j of an ascending list has rows[j] >= first + j, so what an
// entry writes is read by entries up to its own alone.  One wave takes a
// list's K or V (or a slice of SB bytes of each row) from the first entry on
// and has read an entry before it writes it or a later one.
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
    const int64_t first = a.x.first ? a.x.first[s] : 0;
    for (int64_t j0 = lane / L; j0 - lane / L < a.x.count; j0 += U * W) {
        int64_t from[U], to[U];
        chunk_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t j = j0 + u * W, row = j < a.x.count ? rows[j] : -1;
            from[u] = row > first + j ? row_at(a, table, a.b.max_pages, row, g) : -1;
            to[u] = from[u] < 0 ? -1 : row_at(a, table, a.b.max_pages, first + j, g);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (to[u] >= 0) v[u] = *reinterpret_cast<const chunk_t*>(x + from[u]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (to[u] >= 0) *reinterpret_cast<chunk_t*>(x + to[u]) = v[u];
        asm volatile("" ::: "memory");
    }
}

template <int D>
void launch_apart(hipStream_t s, KeepArgs a) {
    constexpr int W = 512 / D, U = 4;
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
// before them, the keep - recent of the largest weights.  Weights become
// 32-bit keys of the same order; four passes over 8 bits each, from the top,
// narrow the key of the last one chosen down (a histogram of 256 bins, 32
// copies apart by lane, so that equal weights do not meet in one LDS word),
// then a pass counts per 64 rows what lies over that key and at it, and a last
// one writes the chosen, of the equal ones the first.

constexpr int EVICT_T = 1024, EVICT_WAVES = EVICT_T / WAVE;
constexpr int EVICT_CELLS = 1024;  // of 64 rows

struct EvictArgs {
    PagedBatch b;
    EvictRows x;
    int kv_heads;
    int64_t max_len;
};

// Ascending with the weight; NaN lowest, the zeros alike.
__device__ inline uint32_t weight_key(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return w != w ? 0u : u >> 31 ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(EVICT_T) void evict_kernel(EvictArgs a) {
    __shared__ uint32_t bins[256 * 32];
    __shared__ uint32_t cells[2 * EVICT_CELLS];
    __shared__ uint32_t sums[EVICT_WAVES], found[2];
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = tid / WAVE;
    const int64_t list = blockIdx.x, s = list / a.kv_heads;
    const float* w = a.x.weights + list * a.x.ldw;
    float* kept = a.x.kept + list * a.x.kept_ld;
    int32_t* rows = a.x.rows + list * a.x.keep;
    const int64_t len = a.b.lens[s], n = len < 0 ? 0 : len < a.max_len ? len : a.max_len;
    const int64_t keep = a.x.keep;
    if (n <= keep) {
        for (int64_t i = tid; i < keep; i += EVICT_T) {
            rows[i] = i < n ? int32_t(i) : -1;
            if (i < n && kept != w) kept[i] = w[i];
        }
        return;
    }
    const int64_t old = n - a.x.recent;
    uint32_t left = uint32_t(keep - a.x.recent);  // to be chosen of the first `old` rows
    uint32_t key = 0xffffffffu;                   // ... over this key, and `left` at it
    if (left) {
        key = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256 * 32; i += EVICT_T) bins[i] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
            constexpr int U = 8;
            for (int64_t i0 = tid; i0 < old; i0 += U * EVICT_T) {
                float x[U];
#pragma unroll
                for (int u = 0; u < U; ++u) x[u] = i0 + u * EVICT_T < old ? w[i0 + u * EVICT_T] : 0.0f;
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t k = weight_key(x[u]);
                    if (i0 + u * EVICT_T < old && (k & mask) == key)
                        atomicAdd(&bins[(k >> shift & 255) * 32 + lane % 32], 1u);
                }
            }
            __syncthreads();
            // Bin b's count in the four threads 4 b .. 4 b + 3; then how many lie
            // over bin b, from the top: a wave has 16 bins.
            uint32_t mine = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine += bins[tid * 8 + i];
            mine += __shfl_xor(mine, 1, WAVE);
            mine += __shfl_xor(mine, 2, WAVE);
            uint32_t above = 0;  // of the wave's bins
            for (int i = 1; i < 16; ++i) {
                const uint32_t o = __shfl(mine, lane + 4 * i, WAVE);
                above += lane / 4 + i < 16 ? o : 0;
            }
            if (lane == 0) sums[wave] = above + mine;
            __syncthreads();
            for (int i = wave + 1; i < EVICT_WAVES; ++i) above += sums[i];
            if (above < left && left <= above + mine && lane % 4 == 0) found[0] = uint32_t(tid / 4), found[1] = above;
            __syncthreads();
            key |= found[0] << shift;
            left -= found[1];
        }
    }
    // Rows over the key and at it, by cells of 64.
    uint32_t over = 0, at = 0;  // before this part
    for (int64_t base = 0; base < old; base += EVICT_CELLS * WAVE) {
        const int64_t end = old - base < EVICT_CELLS * WAVE ? old - base : EVICT_CELLS * WAVE;
        const int ncell = int((end + WAVE - 1) / WAVE);
        for (int c = wave; c < ncell; c += EVICT_WAVES) {
            const int64_t i = base + c * WAVE + lane;
            const uint32_t k = i < old ? weight_key(w[i]) : 0;
            const uint64_t bo = __ballot(i < old && k > key), be = __ballot(i < old && k == key);
            if (lane == 0) cells[2 * c] = __popcll(bo), cells[2 * c + 1] = __popcll(be);
        }
        __syncthreads();
        // Each thread a cell: the counts before it.
        uint32_t o = tid < ncell ? cells[2 * tid] : 0, e = tid < ncell ? cells[2 * tid + 1] : 0;
        uint32_t po = o, pe = e;
        for (int d = 1; d < WAVE; d *= 2) {
            const uint32_t x = __shfl_up(po, d, WAVE), y = __shfl_up(pe, d, WAVE);
            if (lane >= d) po += x, pe += y;
        }
        if (lane == WAVE - 1) bins[2 * wave] = po, bins[2 * wave + 1] = pe;
        __syncthreads();
        uint32_t to = over, te = at;
        for (int i = 0; i < EVICT_WAVES; ++i) {
            if (i < wave) po += bins[2 * i], pe += bins[2 * i + 1];
            to += bins[2 * i], te += bins[2 * i + 1];
        }
        if (tid < ncell) cells[2 * tid] = over + po - o, cells[2 * tid + 1] = at + pe - e;
        __syncthreads();
        // A chosen row's place: the chosen before it.  (In place a weight goes no
        // further down than its own part's rows: each part is read before any
        // of it is written.)
        for (int c0 = 0; c0 < ncell; c0 += 4 * EVICT_WAVES) {
            float x[4];
            int64_t place[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = c0 + u * EVICT_WAVES + wave;
                const int64_t i = base + c * WAVE + lane;
                place[u] = -1;
                if (c >= ncell) continue;
                x[u] = i < old ? w[i] : 0.0f;
                const uint32_t k = weight_key(x[u]);
                const uint64_t before = (uint64_t(1) << lane) - 1;
                const uint64_t bo = __ballot(i < old && k > key), be = __ballot(i < old && k == key);
                const uint32_t no = cells[2 * c] + __popcll(bo & before), ne = cells[2 * c + 1] + __popcll(be & before);
                if (i < old && (k > key || (k == key && ne < left))) place[u] = no + (ne < left ? ne : left);
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (place[u] >= 0) {
                    rows[place[u]] = int32_t(base + (c0 + u * EVICT_WAVES + wave) * WAVE + lane);
                    kept[place[u]] = x[u];
                }
        }
        over = to, at = te;
        __syncthreads();
    }
    // The recent rows, and zeros for the rows to come.
    const int64_t chosen = keep - a.x.recent;
    for (int64_t i0 = 0; i0 < a.x.recent; i0 += EVICT_T) {
        const int64_t i = i0 + tid;
        const float x = i < a.x.recent ? w[old + i] : 0.0f;
        __syncthreads();
        if (i < a.x.recent) rows[chosen + i] = int32_t(old + i), kept[chosen + i] = x;
    }
    __syncthreads();
    for (int64_t i = keep + tid; i < n && i < a.x.kept_ld; i += EVICT_T) kept[i] = 0.0f;
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
    if (b.nseq * kv.kv_heads >= MAX_BLOCKS) fail(E_CAPACITY, "kv_evict: too many lists for one call");
    EvictArgs a{b, x, kv.kv_heads, max_len};
    evict_kernel<<<dim3(unsigned(b.nseq * kv.kv_heads)), dim3(EVICT_T), 0, s>>>(a);
    OMG_HIP(hipGetLastError());
    move_rows(s, kv, b, KeepRows{x.rows, x.keep, x.keep, nullptr, 1, x.to_table, x.to_ld});
}

}  // namespace omg
