// The paged K/V cache: appending rows to it, and the checks that its callers
// share.
#include <string>

#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

// ------------------------------------------------------------------ append
//
// y = x / sqrt(mean(x^2) + eps) * w;  (a, b) -> (a cos - b sin, b cos + a
// sin) for the rotated pairs;  q *= q_scale;  one rounding to the cache's
// type.  Bound by the bytes read and written: 6,200 tokens of 16 256-wide
// heads, f32 to f16, 37 us = 4.1 TB/s; 16,200 of 48 128-wide heads, bf16,
// 82 us = 4.9 TB/s (a copy of 1 GB reaches 4.7); one token each of 12
// sequences 3.8 us, the launch.  A lane holds 8 consecutive
// elements of a head (32-byte f32 loads, 16-byte stores), so a head takes
// HD / 8 lanes and a wave W = 512 / HD heads at once; the partner of a
// half-layout pair sits in another lane of the same head (rope_dims is a
// multiple of 16) and comes by a shuffle.  A wave takes U such sets of one
// token's heads, all loads issued first: four where that leaves enough waves
// for the chip.

template <int L>  // sum over aligned groups of L lanes, the same bits in each
__device__ inline float group_sum(float v) {
    v += dpp_f32<0xb1>(v);
    v += dpp_f32<0x4e>(v);
    v += dpp_f32<0x141>(v);
    if constexpr (L >= 16) v += dpp_f32<0x140>(v);
    if constexpr (L >= 32) v += __shfl_xor(v, 16, WAVE);
    if constexpr (L >= 64) v += __shfl_xor(v, 32, WAVE);
    return v;
}

struct AppendArgs {
    PagedKv kv;
    PagedBatch b;
    KvSource src;
    void* q_out;
    int64_t ldq;
    int nq, nkv;       // head slots: nq queries, nkv keys, nkv values
    int page_shift;
    int items;         // waves per token
};

template <typename S, typename T, int HD, int U>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    constexpr int L = HD / 8, W = WAVE / L;
    const int lane = int(threadIdx.x) % WAVE;
    const int64_t id = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    if (id >= a.b.t * a.items) return;
    const int64_t tok = id / a.items;
    const int item = int(id - tok * a.items);
    const SeqRow at = token_row(a.b, tok, lane);
    if (at.seq < 0) return;  // a row that no sequence has
    const int c0 = (lane % L) * 8;
    const int slots = a.nq + 2 * a.nkv;

    float x[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int slot = (item * U + u) * W + lane / L;
        if (slot < slots) {
            const int h = slot < a.nq ? slot : (slot - a.nq) % (a.nkv ? a.nkv : 1);
            const void* base = slot < a.nq ? a.src.q : slot < a.nq + a.nkv ? a.src.k : a.src.v;
            const int64_t ld = slot < a.nq ? a.src.ld : a.src.ldkv;
            load8(static_cast<const S*>(base) + tok * ld + int64_t(h) * HD + c0, x[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[u][i] = 0.0f;
        }
    }
    // The pairs' (cos, sin) of the lane's elements and its sign in the pair:
    // y' = y cos + sign * partner * sin; outside the pairs elements stay as
    // they are (whole lanes: rope_dims is a multiple of 16).
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
    bool rotated = false;
    const int half = a.src.rope_dims / 2;
    int hop = 0;  // lanes to the partner (half layouts)
    if (a.src.rope) {
        int64_t pos = a.src.positions ? int64_t(a.src.positions[tok]) : a.b.prefix_len + at.row;
        pos = pos < 0 ? 0 : pos >= a.src.rope_rows ? a.src.rope_rows - 1 : pos;
        const float* rt = a.src.rope + pos * a.src.rope_dims;
        if (a.src.rope_layout == 1) {
            if (c0 < a.src.rope_dims) {
                rotated = true;
                float r[8];
                load8(rt + c0, r);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    cs[2 * i] = cs[2 * i + 1] = r[2 * i];
                    sn[2 * i] = -r[2 * i + 1];
                    sn[2 * i + 1] = r[2 * i + 1];
                }
            }
        } else {
            const int apart = a.src.rope_layout == 0 ? half : HD / 2;
            const bool second = c0 >= apart;
            const int i0 = second ? c0 - apart : c0;  // the lane's first pair
            if (i0 < half) {
                rotated = true;
                float r[16];
                load8(rt + 2 * i0, r);
                load8(rt + 2 * i0 + 8, r + 8);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    cs[i] = r[2 * i];
                    sn[i] = second ? r[2 * i + 1] : -r[2 * i + 1];
                }
                hop = second ? -(apart / 8) : apart / 8;
            }
        }
    }
    // The token's cache row; none where its page lies outside the pool.
    int64_t row_off = -1;
    if (a.nkv && at.row >= 0 && (at.row >> a.page_shift) < a.b.max_pages) {
        const int64_t p = a.b.table[at.seq * a.b.table_ld + (at.row >> a.page_shift)];
        if (p >= 0 && p < a.kv.npages)
            row_off = p * a.kv.page_stride + (at.row & (a.kv.page - 1)) * int64_t(HD);
    }

#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int slot = (item * U + u) * W + lane / L;
        const bool is_q = slot < a.nq, is_v = slot >= a.nq + a.nkv;
        const int h = is_q ? slot : (slot - a.nq) % (a.nkv ? a.nkv : 1);
        const float* w = is_q ? a.src.q_norm : is_v ? nullptr : a.src.k_norm;
        if (a.src.q_norm || a.src.k_norm || a.src.v_norm) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += x[u][i] * x[u][i];
            ss = group_sum<L>(ss);
            if (w || (is_v && a.src.v_norm)) {
                const float inv = 1.0f / sqrtf(ss / float(HD) + a.src.eps);
                float g[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = 1.0f;
                if (w) load8(w + c0, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u][i] = x[u][i] * inv * g[i];
            }
        }
        float y[8];  // (an infinite partner times sin 0 would be NaN; choosing y itself: 35 -> 42 us)
        if (a.src.rope_layout == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = x[u][i] * cs[i] + (rotated ? x[u][i ^ 1] : 0.0f) * sn[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float other = __shfl(x[u][i], lane + hop, WAVE);
                y[i] = x[u][i] * cs[i] + (rotated ? other : 0.0f) * sn[i];
            }
        }
        if (slot >= slots) continue;
        if (is_q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= a.src.q_scale;
            store8(static_cast<T*>(a.q_out) + tok * a.ldq + int64_t(h) * HD + c0, y);
        } else if (row_off >= 0) {
            T* dst = static_cast<T*>(is_v ? a.kv.v : a.kv.k) + row_off + int64_t(h) * a.kv.page * HD + c0;
            store8(dst, is_v ? x[u] : y);
        }
    }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int log2_of(int64_t n) {
    int s = 0;
    while ((int64_t(1) << s) < n) ++s;
    return s;
}

void check_kv(const PagedKv& kv, const char* who) {
    const std::string w(who);
    if (kv.dtype != ELEM_F16 && kv.dtype != ELEM_BF16) fail(E_INVALID, w + ": the cache's type must be f16 or bf16");
    if (kv.head_dim != 64 && kv.head_dim != 128 && kv.head_dim != 256 && kv.head_dim != 512)
        fail(E_INVALID, w + ": head_dim must be 64, 128, 256 or 512");
    if (kv.kv_heads <= 0 || kv.kv_heads > 1024) fail(E_INVALID, w + ": kv_heads must be 1 to 1024");
    if (kv.page != 16 && kv.page != 32 && kv.page != 64 && kv.page != 128 && kv.page != 256)
        fail(E_INVALID, w + ": page must be 16, 32, 64, 128 or 256 rows");
    if (kv.npages <= 0 || kv.npages > 0x7fffffff) fail(E_INVALID, w + ": npages out of range");
    const int64_t own = int64_t(kv.kv_heads) * kv.page * kv.head_dim;
    if (kv.page_stride < own || kv.page_stride % 8 || kv.page_stride > (int64_t(1) << 31))
        fail(E_INVALID, w + ": page_stride must hold a page and be a multiple of 8");
    if (!kv.k || !kv.v || !aligned16(kv.k) || !aligned16(kv.v))
        fail(E_INVALID, w + ": k and v must be 16-byte aligned device pointers");
}

void check_batch(const PagedBatch& b, const PagedKv& kv, const char* who) {
    const std::string w(who);
    if (b.nseq <= 0 || b.t <= 0 || b.nseq > (1 << 20) || b.t > (1 << 24))
        fail(E_INVALID, w + ": nseq must be 1 to 2^20 and t 1 to 2^24");
    if (!b.lens || !b.table) fail(E_INVALID, w + ": null lens or table");
    if (!b.start && b.t != b.nseq) fail(E_INVALID, w + ": without start every sequence has one token (t = nseq)");
    if (b.max_pages <= 0 || b.max_pages > 0x3fffffff / kv.page || b.table_ld < b.max_pages)
        fail(E_INVALID, w + ": max_pages out of range or past table_ld");
    if (b.prefix_len < 0 || b.prefix_len > 0x3fffffff) fail(E_INVALID, w + ": prefix_len out of range");
    if (b.prefix_len > 0 && !b.prefix_table) fail(E_INVALID, w + ": null prefix_table");
}

namespace {

template <typename S, typename T, int HD>
void append_hd(hipStream_t s, AppendArgs a) {
    constexpr int W = 512 / HD;
    const int slots = a.nq + 2 * a.nkv;
    const int sets = (slots + W - 1) / W;
    const auto blocks = [&](int u) {
        a.items = (sets + u - 1) / u;
        const int64_t n = (a.b.t * a.items + 3) / 4;
        if (n >= MAX_BLOCKS) fail(E_CAPACITY, "kv_append: too many rows for one call");
        return unsigned(n);
    };
    if (sets < 4 || a.b.t * sets <= 8192) {
        const unsigned n = blocks(1);
        kv_append_kernel<S, T, HD, 1><<<dim3(n), dim3(256), 0, s>>>(a);
    } else {
        const unsigned n = blocks(4);
        kv_append_kernel<S, T, HD, 4><<<dim3(n), dim3(256), 0, s>>>(a);
    }
    OMG_HIP(hipGetLastError());
}

template <typename S, typename T>
void append_types(hipStream_t s, const AppendArgs& a) {
    switch (a.kv.head_dim) {
        case 64: return append_hd<S, T, 64>(s, a);
        case 128: return append_hd<S, T, 128>(s, a);
        case 256: return append_hd<S, T, 256>(s, a);
        default: return append_hd<S, T, 512>(s, a);
    }
}

}  // namespace

void launch_kv_append(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const KvSource& src, void* q_out,
                      int64_t ldq) {
    check_kv(kv, "kv_append");
    check_batch(b, kv, "kv_append");
    if (src.dtype != ELEM_F32 && src.dtype != kv.dtype)
        fail(E_INVALID, "kv_append: the source must be f32 or the cache's type");
    const int per16 = src.dtype == ELEM_F32 ? 4 : 8;
    if (!src.q && !src.k) fail(E_INVALID, "kv_append: neither queries nor keys");
    if (!src.k != !src.v) fail(E_INVALID, "kv_append: keys and values come together");
    if (!aligned16(src.q) || !aligned16(src.k) || !aligned16(src.v) || !aligned16(q_out))
        fail(E_INVALID, "kv_append: pointers must be 16-byte aligned");
    if (src.q) {
        if (src.heads <= 0 || src.heads > 4096) fail(E_INVALID, "kv_append: heads must be 1 to 4096");
        if (!q_out) fail(E_INVALID, "kv_append: null q_out");
        const int64_t width = int64_t(src.heads) * kv.head_dim;
        if (src.ld < width || src.ld % per16 || ldq < width || ldq % 8)
            fail(E_INVALID, "kv_append: ld and ldq must hold the heads and be whole 16 bytes");
    }
    if (src.k && (src.ldkv < int64_t(kv.kv_heads) * kv.head_dim || src.ldkv % per16))
        fail(E_INVALID, "kv_append: ldkv must hold the heads and be whole 16 bytes");
    if (src.rope) {
        if (src.rope_rows <= 0) fail(E_INVALID, "kv_append: empty rope table");
        if (src.rope_dims <= 0 || src.rope_dims > kv.head_dim || src.rope_dims % 16)
            fail(E_INVALID, "kv_append: rope_dims must be a multiple of 16 up to head_dim");
        if (src.rope_layout < 0 || src.rope_layout > 2) fail(E_INVALID, "kv_append: unknown rope layout");
        if (!aligned16(src.rope)) fail(E_INVALID, "kv_append: pointers must be 16-byte aligned");
    }
    if (!aligned16(src.q_norm) || !aligned16(src.k_norm))
        fail(E_INVALID, "kv_append: pointers must be 16-byte aligned");
    AppendArgs a{kv, b, src, q_out, ldq, src.q ? src.heads : 0, src.k ? kv.kv_heads : 0, log2_of(kv.page), 0};
    if (!src.rope) a.src.rope_layout = 0, a.src.rope_dims = 0;
    if (kv.dtype == ELEM_F16)
        src.dtype == ELEM_F32 ? append_types<float, half_t>(s, a) : append_types<half_t, half_t>(s, a);
    else
        src.dtype == ELEM_F32 ? append_types<float, bf16_t>(s, a) : append_types<bf16_t, bf16_t>(s, a);
}

}  // namespace omg
