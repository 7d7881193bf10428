// Attention over a prefix that all sequences of a batch share and over each
// sequence's own rows, both on pages of a K/V pool:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c (s_j - m) + lift),  s_j = q . k_j,
// c = scale log2(e), m a running maximum of s, over the keys j that the
// query sees.  Partial results over ranges of keys are their means sum p v /
// sum p and lg = log2 of the ranges' sums of 2^(c s): out is the means' mean
// with the weights 2^(lg - max lg).  (Sums of bf16 values may pass f32's
// largest, means do not.)
//
// Queries are rows (token, head) of one KV head, so that a tile of rows
// takes every key and value it reads once for all of them: tiles of the
// prefix hold rows of any sequences, tiles of a sequence's own keys its rows
// alone.  Where sequences bring at least a wave of rows each (prompts,
// questions) a tile runs through the prefix and then through the own keys
// of the sequences it holds (`fused`); where they bring a few (a step of
// decoding) the own keys have work items of their own, in the same launch.
// Few tiles split the keys over work items; attention_join joins these.
//
// MASKED (tree_attention.hip): of its sequence's new rows a token sees those
// that its mask has bits for; the lengths' order says nothing about these.
//
// Tiles (MFMA shape = rows of a wave x keys):
//   WAVES_32:   4 waves x 32 rows, 32-key K and V tiles shared in LDS, two
//               buffers, the next tile's loads in flight (four buffers, and
//               with them one workgroup a CU: 62 us where two take 42);
//   WAVES_16:   4 waves x 16 rows, the same (few rows; head_dim 512, whose
//               tiles are 16 keys long);
//   WAVES_KEYS: 16 rows, each wave takes every fourth 16-key tile into LDS
//               of its own; the waves join through LDS at the end.
// Both products leave the query in the lane: S^T = K Q^T with the lane's
// query as column, then O^T += V^T P^T, whose P^T operand is the lane's own
// scores; V^T comes from row-major V by LDS transposing reads of 4 keys.
//
// K and V tiles come by buffer loads to LDS, 16 bytes a lane, from a
// resource that ends with the last valid row of the page (rows behind it
// and pages outside the pool arrive as zeros, so that nothing they hold
// meets a probability of zero).  The 16-byte chunks of a row are XORed with
// bits of its number, so that half a wave's reads fall on distinct banks: K's
// 16 rows x 16 bytes, V's 4 rows x 64 bytes or 8 x 32 (counted: none meet).
//
// Measured, and what bounds it:
//   questions, 6,300 tokens x 8 heads of 256 on 8,000 keys (f16): 460-500 us,
//     830-900 TFLOP/s of the 1,190 that a product of 8,192^3 reaches.  392
//     tiles on 512 places; MFMAs take 45 % of the busy CUs' cycles, other
//     vector instructions 33 %, LDS 22 %: a tile is one chain of dependent
//     steps with two waves a SIMD to fill it, registers allow no third (256
//     vector registers, 4 spilled).
//   64 answers' tokens x 32 heads of 128 on 65,521 shared and 131,000 own
//     keys (bf16): 153 us, 4.4 TB/s: the bytes.
//   208 answers' tokens x 8 heads of 256 on 8,000 keys: 38 + 8 us: 256 items
//     of 16 tiles, the same chain (2.5 us a tile), and 29 MB of partials.
//   12 answers' tokens x 4 heads of 256 on 2,000 keys: 8.5 + 4 us: latency.
//   questions, 470 tokens x 8 heads of 512 on 2,000 keys (bf16): 43 + 12 us:
//     61 MB of partials written and read.
//   208 answers' tokens x 8 heads of 512 on 8,000 keys (f16): 100 us: one
//     workgroup a CU, by the own items' 128 KiB of LDS.
//   A window shortens work items and does not lessen them: of the 208 answers'
//     prefix splits most have nothing to do at a window of 512, 46 -> 32 us;
//     64 answers on 65,521 keys at 1,024 154 -> 66 us; the 6,300 questions'
//     tokens, whose items are not split, at 512 480 -> 61 us.
#pragma once

#include <algorithm>
#include <atomic>
#include <climits>
#include <string>

#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

namespace {

enum Tile { WAVES_KEYS = 0, WAVES_16 = 1, WAVES_32 = 2 };

// The running maximum may lag by LAG binary orders in p.  For f16 all p stand
// 7 orders higher: the largest lie in 2^7 .. 2^15, so that f16 holds p with
// all its bits down to 2^-21 of the largest, and those below to 2^-32 of it
// (without: 60,000 keys of 2^-20.5 each 4 % off).  bf16 has f32's exponents,
// and values that leave its sums no room to be lifted.  A smaller lag takes
// the outputs' products with 2^(c (m - m')) more often: 4 orders 530 us for
// the questions above, 8 480.
constexpr float LAG = 8.0f;
template <typename T>
constexpr float lift = std::is_same_v<T, half_t> ? 7.0f : 0.0f;

struct Plan {
    int tile;       // Tile of the prefix / fused items
    bool fused;     // own keys in the prefix items' tiles
    bool whole;     // fused and not split: prefix and own keys in one item
    int ntile, np, chunk_p;            // prefix: row tiles, splits, keys per split
    int64_t own_tiles;                 // bound of the sequences' 16-row tiles (not fused)
    int os, chunk_o;                   // own keys: splits, keys per split
    __host__ __device__ int64_t slots() const { return whole ? 1 : np + os; }
};

struct Args {
    PagedKv kv;
    PagedBatch b;
    SharedAttn x;
    Plan p;
    int hpg, page_shift;
    int64_t max_len;           // rows a table reaches
    int64_t prefix_blocks;     // (a multiple of 8)
    float c;                   // scale log2(e)
    TreeMask tree;             // (MASKED)
    float* part_o;             // [slots][t * heads][head_dim], null: results go out
    float* part_lg;            // [slots][t * heads]
};

typedef __attribute__((address_space(3))) void* lds_ptr;
typedef short short4v __attribute__((ext_vector_type(4)));

__device__ inline floatx16 mfma32(half8 a, half8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx16 mfma32(bf16x8 a, bf16x8 b, floatx16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma16(half8 a, half8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
__device__ inline floatx4 mfma16k16(half4 a, half4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma16k16(bf16x4 a, bf16x4 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(short4v, a), __builtin_bit_cast(short4v, b), c,
                                                     0, 0, 0);
}

template <typename T, int D, int TILE>
struct Core {
    static constexpr int RW = TILE == WAVES_32 ? 32 : 16;                    // rows of a wave
    static constexpr int KT = TILE == WAVES_KEYS || D == 512 ? 16 : 32;      // keys of a tile
    static constexpr int KS = RW == 32 ? 16 : 32;              // head dims per MFMA of K Q^T
    static constexpr int NS = D / KS, NC = D / RW;
    static constexpr int NB = KT / RW < 1 ? 1 : KT / RW;       // score blocks
    static constexpr int SR = RW == 32 ? 16 : 4;               // scores of a lane per block
    static constexpr int CH = D / 8;                           // 16-byte chunks of a row
    typedef typename Vec8<T>::type frag;
    typedef std::conditional_t<RW == 32, floatx16, floatx4> acc;

    frag q[NS];
    acc o[NC];
    float m, l;  // running maximum of the raw scores; the lane's share of sum p

    // The chunks of row r are XORed with these (sums of r's bits, so that an
    // address follows from others): 256 bytes are one turn over the banks.
    static __device__ int swz_k(int row) { return CH >= 16 ? row & 15 : row >> 1 & 7; }
    static __device__ int swz_v(int row) {
        return CH < 16 ? (row & 3) << 1 : RW == 32 ? (row & 3) << 2 : (row & 7) << 1;
    }
    static __device__ float row_max(float v) {
        if constexpr (RW == 32) {
            const uint32_t u = __builtin_bit_cast(uint32_t, v);
            const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            return fmaxf(__builtin_bit_cast(float, uint32_t(p[0])), __builtin_bit_cast(float, uint32_t(p[1])));
        } else {
            return max_lanes_16_32(v);
        }
    }
    static __device__ float row_sum(float v) {
        if constexpr (RW == 32) {
            const uint32_t u = __builtin_bit_cast(uint32_t, v);
            const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
            return __builtin_bit_cast(float, uint32_t(p[0])) + __builtin_bit_cast(float, uint32_t(p[1]));
        } else {
            return sum_lanes_16_32(v);
        }
    }

    __device__ void init(const T* row, int lane) {
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            frag z{};
            q[s] = row ? *reinterpret_cast<const frag*>(row + s * KS + 8 * (lane / RW)) : z;
        }
#pragma unroll
        for (int i = 0; i < NC; ++i)
#pragma unroll
            for (int r = 0; r < SR; ++r) o[i][r] = 0.0f;
        m = -INFINITY;
        l = 0.0f;
    }

    // The lane's addresses in a tile, in bytes: of its K operands' first chunk
    // (the chunk of step st XORed in: its bits are apart from the row's) and
    // of its V reads.  They are hidden from the compiler in each tile, which
    // would keep all their XORs in registers otherwise: 24 of 256, and no
    // room left to read operands ahead.
    static __device__ uint32_t k_base(int lane) {
        const int row = lane % RW;
        return uint32_t(row * D * 2 + ((lane / RW) ^ swz_k(row)) * 16);
    }
    static __device__ uint32_t v_base(int lane) {
        const int i16 = lane % 16, g16 = lane / 16;
        const int row = (RW == 32 ? 4 * (g16 / 2) : 4 * g16) + i16 / 4;
        const int ch = (RW == 32 ? 2 * (g16 % 2) : 0) + (i16 % 4) / 2;
        return uint32_t(row * D * 2 + (ch ^ swz_v(row)) * 16 + (i16 % 2) * 8);
    }
    // V rows r .. r + 3 of the lane's 16-lane group, one column a lane: lane i
    // of the group gives the address of row i / 4, columns 4 (i % 4) .. + 3
    // and gets column i of the four rows.
    static __device__ short4v read_tr(uint32_t at, int offset) {
        typedef __attribute__((address_space(3))) short4v* ptr;
        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)(at + offset));
    }
    static __device__ frag read_k(uint32_t at, int offset) {
        typedef __attribute__((address_space(3))) frag* ptr;
        return *(ptr)(uintptr_t)(at + offset);
    }

    // One tile at LDS address `at` (K, then V) whose first key is k0; the
    // lane's query sees the keys lo .. hi - 1 that are not in `bad` (a bit
    // per key of the tile).
    __device__ void tile(uint32_t at, int lane, int k0, bool full, int lo, int hi, uint32_t bad, float c) {
        acc s[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < SR; ++r) s[j][r] = 0.0f;
        uint32_t ka = at + k_base(lane), va = at + KT * D * 2 + v_base(lane);
        asm volatile("" : "+v"(ka), "+v"(va));
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const frag kf = read_k(ka ^ uint32_t(st * (KS / 8) * 16), j * RW * D * 2);
                if constexpr (RW == 32)
                    s[j] = mfma32(kf, q[st], s[j]);
                else
                    s[j] = mfma16(kf, q[st], s[j]);
            }
        pipeline<NS * NB, 1, 1>();
        // The first V operands go out ahead of the softmax, which hides them.
        frag vf[VA];
#pragma unroll
        for (int i = 0; i < VA; ++i) vf[i] = read_v(va, i);
        __builtin_amdgcn_sched_barrier(0);
        if (!full) {
            // (the lane's keys: a constant of (j, r) past k0 + 4 * its group)
            const int first = k0 + 4 * (lane / RW), from = lo - first, to = hi - first;
            const uint32_t out = bad >> (4 * (lane / RW));
#pragma unroll
            for (int j = 0; j < NB; ++j)
#pragma unroll
                for (int r = 0; r < SR; ++r) {
                    const int kk = RW == 32 ? 8 * (r / 4) + r % 4 : 16 * j + r;
                    const bool see = kk >= from && kk < to && !(out & (1u << kk));
                    s[j][r] = see ? s[j][r] : -INFINITY;
                }
        }
        float mt = s[0][0];
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < SR; ++r) mt = fmaxf(mt, s[j][r]);
        mt = row_max(mt);
        // The maximum moves where a row's scores pass it by more than LAG.
        if (__any((mt - m) * c > LAG || (m == -INFINITY && mt > m))) {
            const float mn = fmaxf(m, mt);
            const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * c);
            m = mn;
            l *= al;
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int r = 0; r < SR; ++r) o[i][r] *= al;
        }
        const float mc = m == -INFINITY ? 0.0f : m * c - lift<T>;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int r = 0; r < SR; ++r) {
                const float p = __builtin_amdgcn_exp2f(fmaf(s[j][r], c, -mc));
                s[j][r] = p;
                sum += p;
            }
        l += sum;
        // P^T operands: the lane's scores of each MFMA step over the keys.
        frag pf[VS];
#pragma unroll
        for (int j = 0; j < VS; ++j)
#pragma unroll
            for (int r = 0; r < (KT == 16 ? 4 : 8); ++r)
                pf[j][r] = T(RW == 32 ? s[0][8 * j + r] : s[r / 4][r % 4]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < NC * VS; ++i) {
            const frag v = vf[i % VA];
            if (i + VA < NC * VS) vf[i % VA] = read_v(va, i + VA);
            if constexpr (RW == 32) {
                o[i / VS] = mfma32(v, pf[i % VS], o[i / VS]);
            } else if constexpr (KT == 32) {
                o[i] = mfma16(v, pf[0], o[i]);
            } else {
                typedef T frag4 __attribute__((ext_vector_type(4)));
                const frag4 a = {v[0], v[1], v[2], v[3]}, b = {pf[0][0], pf[0][1], pf[0][2], pf[0][3]};
                o[i] = mfma16k16(a, b, o[i]);
            }
        }
        pipeline<NC * VS, KT == 16 ? 1 : 2, 0>();
    }
    // V^T operand i: head dims i / VS, keys of step i % VS.
    static constexpr int VS = RW == 32 ? 2 : 1;      // MFMA steps over the keys
    static constexpr int VA = 4;                     // operands read ahead
    static __device__ frag read_v(uint32_t va, int i) {
        union {
            short4v h[2];
            frag f;
        } v;
        if constexpr (RW == 32) {
            const uint32_t a = va ^ uint32_t(i / 2 * 64);
            v.h[0] = read_tr(a, 16 * (i % 2) * D * 2);
            v.h[1] = read_tr(a, (16 * (i % 2) + 8) * D * 2);
        } else {
            const uint32_t a = va ^ uint32_t(i * 32);
            v.h[0] = read_tr(a, 0);
            if constexpr (KT == 32)
                v.h[1] = read_tr(a, 16 * D * 2);
            else
                v.h[1] = v.h[0];
        }
        return v.f;
    }
    // The order of a run of N MFMAs, each on an operand of READS LDS reads:
    // VA operands' reads go first where FIRST, then one operand's after each
    // MFMA.  (Left alone, the compiler reads one operand and waits for it.)
    template <int N, int READS, int FIRST>
    static __device__ void pipeline() {
        if constexpr (FIRST) __builtin_amdgcn_sched_group_barrier(0x100, VA * READS, 0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (i + VA < N) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        }
    }
    // The lane's four consecutive head dims of output quad (i, rr).
    static constexpr int QUADS = SR / 4;
    static __device__ int dim_of(int lane, int i, int rr) {
        return RW == 32 ? 32 * i + 8 * rr + 4 * (lane / 32) : 16 * i + 4 * (lane / 16);
    }
};

// log2 of a row's sum of 2^(c s), from its c m - lift and l.
__device__ inline float log_sum(float cm, float l) { return l == 0.0f ? -INFINITY : cm + __builtin_amdgcn_logf(l); }

// A mean of values of T in T.  p is rounded for its product with V and not in
// l (lse has all of l's bits; the rounded p's sum beside it, a register more,
// took 46 -> 49 us for the 208 answers' tokens above), so the mean of values
// near T's largest may come out a step past it: it is no larger than they are.
template <typename T>
__device__ inline T mean(float x) {
    const float most = std::is_same_v<T, half_t> ? 65504.0f : 3.3895314e38f;
    return T(fabsf(x) < INFINITY ? fminf(fmaxf(x, -most), most) : x);
}

// Where a row's result of slot `slot` goes: the partials, or the output.
template <typename T>
struct Sink {
    const Args& a;
    int64_t row;    // tok * heads + head
    int64_t out;    // tok * ldo + head * D
    int64_t slot;
    __device__ void stats(float lg) const {
        if (a.part_o)
            a.part_lg[slot * a.b.t * a.x.heads + row] = lg;
        else if (a.x.lse)
            a.x.lse[row] = lg * 0.69314718055994531f;
    }
    // Four elements of the mean (`some`: the row sees a key here).
    template <int D>
    __device__ void quad(int dim, float4 v, bool some) const {
        if (a.part_o) {
            if (some) *reinterpret_cast<float4*>(a.part_o + (slot * a.b.t * a.x.heads + row) * D + dim) = v;
        } else {
            typedef T vec4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<vec4*>(static_cast<T*>(a.x.out) + out + dim) = vec4{mean<T>(v.x), mean<T>(v.y), mean<T>(v.z), mean<T>(v.w)};
        }
    }
};
__device__ inline float4 times(float4 v, float f) { return make_float4(v.x * f, v.y * f, v.z * f, v.w * f); }

// A value that is the same in every lane, in a scalar register.
__device__ inline int uni(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline uint64_t uni_ptr(const void* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return uint64_t(uint32_t(uni(int(uint32_t(v >> 32))))) << 32 | uint32_t(uni(int(uint32_t(v))));
}

constexpr int NW = 4;

// The keys of one work item's segments, tile by tile, through LDS.
template <typename T, int D, int TILE>
struct Stream {
    typedef Core<T, D, TILE> C;
    static constexpr bool KEYS = TILE == WAVES_KEYS;
    static constexpr int KT = C::KT;
    static constexpr int TILE_ELEMS = KT * D;
    static constexpr int INS = TILE_ELEMS * 2 / 1024 / (KEYS ? 1 : NW);  // 1 KiB loads per wave for K, and for V
    static_assert(INS >= 1, "a wave loads at least 1 KiB of a tile");

    static constexpr int NBUF = KEYS ? 1 : 2;

    const Args& a;
    int g, wave, lane;
    T* smem;  // KEYS: [wave][K, V], else [NBUF][K, V]

    __device__ T* buf(int which) const { return smem + (KEYS ? wave : which) * 2 * TILE_ELEMS; }

    // One 1 KiB piece holds RPI rows; the lane's byte offsets in the first
    // piece, from which the others' follow (their rows' bits are apart).
    static constexpr int RPI = 512 / D;
    __device__ void issue(int k0, int klim, T* dst, int p0, int p1) const {
        // A wave's rows lie in one 16-row half of the tile, so in one page.
        const int hf = !KEYS && KT == 32 && wave >= NW / 2 ? 1 : 0;
        const int p = hf ? p1 : p0, kk = k0 + 16 * hf;
        const bool ok = unsigned(p) < unsigned(a.kv.npages);
        int rows = klim - kk;
        rows = rows < 0 ? 0 : rows > 16 ? 16 : rows;
        const int bytes = uni(ok ? rows * D * 2 : 0);
        const int64_t off = 2 * ((ok ? p : 0) * a.kv.page_stride + (int64_t(g) * a.kv.page + (kk & (a.kv.page - 1))) * D);
        const __amdgpu_buffer_rsrc_t rk = rsrc(a.kv.k, off, bytes), rv = rsrc(a.kv.v, off, bytes);
        const int row = (KEYS ? 0 : wave * INS * RPI) + lane / C::CH, pc = lane % C::CH;
        uint32_t ko = uint32_t((row & 15) * D * 2 + (pc ^ C::swz_k(row)) * 16);
        uint32_t vo = uint32_t((row & 15) * D * 2 + (pc ^ C::swz_v(row)) * 16);
        asm volatile("" : "+v"(ko), "+v"(vo));
        T* to = dst + (KEYS ? 0 : wave * INS) * 512;
#pragma unroll
        for (int i = 0; i < INS; ++i) {
            const int r = i * RPI;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_ptr)(to + i * 512), 16, ko ^ uint32_t(C::swz_k(r) * 16),
                                                     r * D * 2, 0, 0);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_ptr)(to + TILE_ELEMS + i * 512), 16,
                                                     vo ^ uint32_t(C::swz_v(r) * 16), r * D * 2, 0, 0);
        }
    }
    static __device__ __amdgpu_buffer_rsrc_t rsrc(const void* base, int64_t off, int bytes) {
        return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(uni_ptr(static_cast<const char*>(base) + off)),
                                                 (short)0, bytes, 0x00020000);
    }

    // Keys kb .. ke - 1 (kb a multiple of 32; rows from klim on do not
    // exist) on the pages table[0 .. plast]; the lane's query sees [lo, hi).
    // Every wave of the workgroup calls it with the same kb and ke.
    // MASKED: of the keys from `base` on, those that the mask of the lane's
    // row (`at`) has.
    template <bool MASKED = false>
    __device__ void run(C& core, const int32_t* table, int plast, int kb, int ke, int klim, bool valid, int lo,
                        int hi, int base = 0, int at = 0) const {
        kb = uni(kb), ke = uni(ke), klim = uni(klim), base = uni(base);
        // (asked for a tile ahead, like its page)
        auto hidden = [&](int k) { return MASKED && valid && k + KT > base ? ~a.tree.seen(at / a.x.heads, k - base) : 0u; };
        const int step = KEYS ? NW * KT : KT;
        int k0 = kb + (KEYS ? wave * KT : 0);
        const int shift = a.page_shift;
        auto fetch = [&](int k) {  // lane 0: the page of key k, lane 1: of key k + 16
            const int i = (k + 16 * (lane & 1)) >> shift;
            return table[i > plast ? plast : i];
        };
        if (k0 >= ke) return;  // (no barrier below where waves differ in k0)
        if constexpr (KEYS) {
            for (int pn = fetch(k0); k0 < ke; k0 += step) {
                const int p = __builtin_amdgcn_readlane(pn, 0);
                if (k0 + step < ke) pn = fetch(k0 + step);
                issue(k0, klim, buf(0), p, p);
                const uint32_t hide = hidden(k0);
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                use<MASKED>(core, buf(0), k0, valid, lo, hi, bad_keys(p, p) | hide);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            }
        } else {
            // The next tile is under way during a tile; its page is asked for
            // before the loads of the tile before it.  (Through the scalar
            // cache every LDS wait would wait for the page too.)
            int pn = fetch(kb), which = 0;
            __syncthreads();  // the buffers may still be read for the segment before
            int p0 = __builtin_amdgcn_readlane(pn, 0), p1 = __builtin_amdgcn_readlane(pn, 1);
            pn = fetch(kb + KT);
            issue(kb, klim, buf(0), p0, p1);
            uint32_t next = hidden(kb);
            for (; k0 < ke; k0 += KT, which ^= 1) {
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                // Every wave's part of the tile has landed, and every wave is
                // done with the other buffer, which is loaded next.
                __syncthreads();
                const uint32_t bad = bad_keys(p0, KT == 32 ? p1 : p0) | next;
                if (k0 + KT < ke) {
                    next = hidden(k0 + KT);
                    p0 = __builtin_amdgcn_readlane(pn, 0), p1 = __builtin_amdgcn_readlane(pn, 1);
                    pn = fetch(k0 + 2 * KT);
                    issue(k0 + KT, klim, buf(which ^ 1), p0, p1);
                }
                use<MASKED>(core, buf(which), k0, valid, lo, hi, bad);
            }
        }
    }
    // The keys of a tile on pages outside the pool.
    __device__ uint32_t bad_keys(int p0, int p1) const {
        const uint32_t n = uint32_t(a.kv.npages);
        return (unsigned(p0) < n ? 0u : 0xffffu) | (unsigned(p1) < n ? 0u : 0xffff0000u);
    }
    // (MASKED: `bad` is a lane's own)
    template <bool MASKED>
    __device__ void use(C& core, const T* tile, int k0, bool valid, int lo, int hi, uint32_t bad) const {
        if (!__ballot(valid && lo < k0 + KT && hi > k0)) return;
        bool full;
        if constexpr (MASKED)
            full = __all(!valid || (bad == 0 && lo <= k0 && hi >= k0 + KT));
        else
            full = bad == 0 && __all(!valid || (lo <= k0 && hi >= k0 + KT));
        core.tile(uint32_t(uintptr_t((lds_ptr)tile)), lane, k0, full, lo, hi, bad, a.c);
    }
};

__device__ inline int imin(int a, int b) { return a < b ? a : b; }
__device__ inline int imax(int a, int b) { return a > b ? a : b; }

// The first key that the window of a query at row `own` behind `prefix` rows
// leaves (own is below zero where a length is short of its sequence's tokens:
// sums that saturate, one instruction each).
__device__ inline int first_seen(int prefix, int own, int window) {
    return window > 0 ? imax(0, __builtin_elementwise_sub_sat(__builtin_elementwise_add_sat(prefix, own), window - 1)) : 0;
}

// A lane's query row.
struct Row {
    bool valid;
    int at;        // tok * heads + head (one register: the tiles need all others)
    int seq, own;  // own: its row in the sequence's cache rows (MASKED: its position behind the prefix)
};

// The first of the cache rows of a sequence's new tokens (below zero where
// its length is short of them).
__device__ inline int own_base(const Args& a, int64_t s) {
    return imax(a.b.lens[s], 0) - (a.b.start ? a.b.start[s + 1] - a.b.start[s] : 1);
}

// The keys of a work item: prefix rows [pb, pe), own rows [ob, oe).
struct Keys {
    int g, pb, pe, ob, oe;
};

// In a tile a key that a query does not see has p = 0, which leaves nothing
// of its values unless these are infinite or NaN, and a sum of finite bf16
// values may pass f32's largest where their mean does not.  Sums that are not
// finite are therefore taken again from the keys their row sees and no
// others, with probabilities that add up to one: `rows` holds a bit per lane
// whose row it is (with log sum lg); a wave writes the quads of head dims it
// has (quarter < 0: all).  A row whose scores hold a NaN has it in lg, and in
// its outputs as they are.
//   A wave takes its rows one after another and a row's keys four at a time,
// until every element is NaN: 0.3 to 0.4 us a key and row.  One infinite
// value in a prefix of 8,000 keys, which all rows see: 208 answers' tokens x 8
// heads of 256 45 us -> 4.4 ms, 6,300 questions' tokens 0.5 -> 111 ms.
//   `walk(lane of a row, keys)` calls keys(from, to, page) for each run of keys
// that the row sees: key k is row k % page length of page(k), which is outside
// the pool where the row does not see it.
template <typename T, int D, typename W>
__device__ void seen_alone(const Args& a, int g, const Row& r, uint64_t rows, float lg, int lane, int64_t slot,
                           int quarter, W walk) {
    constexpr int NQ = D / 4, E = (NQ + WAVE - 1) / WAVE;
    typedef T vec4 __attribute__((ext_vector_type(4)));
#pragma unroll 1
    for (; rows; rows &= rows - 1) {
        const int i = __builtin_ctzll(rows);
        const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
        const auto off = [&](float v) { return __builtin_bit_cast(float, of(__builtin_bit_cast(int, v))); };
        const int at = of(r.at);
        const int64_t tok = at / a.x.heads;
        const int head = at % a.x.heads;
        const float row_lg = off(lg), ref = row_lg == -INFINITY ? 0.0f : row_lg;
        float4 q[E], o[E];
        const auto load = [&](const void* p, int64_t at, float4* x) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                vec4 v{};
                if (lane + e * WAVE < NQ) v = reinterpret_cast<const vec4*>(static_cast<const T*>(p) + at)[lane + e * WAVE];
                x[e] = make_float4(float(v[0]), float(v[1]), float(v[2]), float(v[3]));
            }
        };
        load(a.x.q, tok * a.x.ldq + int64_t(head) * D, q);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float total = 0.0f;  // of the probabilities: one, but for rounding
        bool lost = false;   // every element is NaN, and stays so
        const auto keys = [&](int from, int to, auto page_of) {
            constexpr int U = 4;  // keys under way together
#pragma unroll 1
            for (int k = from; k < to && !lost; k += U) {
                int64_t key[U];
                bool ok[U];
                float4 x[U][E];
                float p[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t page = page_of(imin(k + u, to - 1));
                    ok[u] = k + u < to && page >= 0 && page < a.kv.npages;
                    key[u] = ok[u] ? page * a.kv.page_stride + (int64_t(g) * a.kv.page + ((k + u) & (a.kv.page - 1))) * D : 0;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) load(a.kv.k, key[u], x[u]);
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    float s = 0.0f;
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        s += x[u][e].x * q[e].x + x[u][e].y * q[e].y + x[u][e].z * q[e].z + x[u][e].w * q[e].w;
                    p[u] = __builtin_amdgcn_exp2f(fmaf(wave_sum(s), a.c, -ref));
                    total += ok[u] ? p[u] : 0.0f;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) load(a.kv.v, key[u], x[u]);
                bool nan = true;
#pragma unroll
                for (int e = 0; e < E; ++e) {
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        if (!ok[u]) continue;
                        o[e].x += p[u] * x[u][e].x, o[e].y += p[u] * x[u][e].y;
                        o[e].z += p[u] * x[u][e].z, o[e].w += p[u] * x[u][e].w;
                    }
                    nan = nan && (lane + e * WAVE >= NQ || (o[e].x != o[e].x && o[e].y != o[e].y && o[e].z != o[e].z &&
                                                            o[e].w != o[e].w));
                }
                lost = __all(nan);
            }
        };
        walk(i, keys);
        const Sink<T> out{a, at, tok * a.x.ldo + int64_t(head) * D, slot};
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int c4 = lane + e * WAVE;
            if (c4 < NQ && (quarter < 0 || c4 % 16 / 4 == quarter))
                out.template quad<D>(4 * c4, times(o[e], inv), row_lg != -INFINITY);
        }
    }
}

// The keys of an item that the row of lane i sees.
template <bool MASKED, typename F>
__device__ inline void seen_keys(const Args& a, const Keys& in, const Row& r, int i, F keys) {
    const auto of = [&](int v) { return __builtin_amdgcn_readlane(v, i); };
    const int P = int(a.b.prefix_len), w = a.x.window, seq = of(r.seq), own = of(r.own), plast = (P - 1) >> a.page_shift;
    const int64_t tok = of(r.at) / a.x.heads;
    keys(imax(in.pb, first_seen(P, own, w)), in.pe,
         [&](int k) { return int64_t(a.b.prefix_table[imin(k >> a.page_shift, plast)]); });
    const int base = MASKED ? own_base(a, seq) : 0;
    const int32_t* table = a.b.table + seq * a.b.table_ld;
    keys(imax(in.ob, MASKED ? imin(first_seen(0, own, w), imax(base, 0)) : first_seen(0, own, w)),
         MASKED ? imin(in.oe, a.b.lens[seq]) : imin(in.oe, own + 1), [&](int k) -> int64_t {
             if (MASKED && k >= base && !(a.tree.seen(tok, k - base) & 1)) return -1;
             return table[imin(k >> a.page_shift, int(a.b.max_pages) - 1)];
         });
}

// The results of a wave's rows (not KEYS).  `alone(rows, lg)` takes those again
// whose sums are not finite.
template <typename T, int D, int TILE, typename F>
__device__ inline void emit(const Args& a, Core<T, D, TILE>& core, const Row& r, int lane, int64_t slot, F alone) {
    typedef Core<T, D, TILE> C;
    const float l = C::row_sum(core.l), inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float lg = log_sum(core.m * a.c - lift<T>, l);
    const Sink<T> out{a, r.at, r.at / a.x.heads * a.x.ldo + int64_t(r.at % a.x.heads) * D, slot};
    if (r.valid && lane < C::RW) out.stats(lg);
    float z[4] = {};  // (NaN where a sum is not finite)
#pragma unroll
    for (int i = 0; i < C::NC; ++i)
#pragma unroll
        for (int e = 0; e < C::SR; ++e) z[e % 4] = fmaf(core.o[i][e], 0.0f, z[e % 4]);
    uint64_t bad = __ballot(r.valid && l == l && !(z[0] + z[1] + z[2] + z[3] == 0.0f));
    bad |= bad >> 32;
    if constexpr (C::RW == 16) bad |= bad >> 16;
    bad &= (uint64_t(1) << C::RW) - 1;
    if (r.valid && !(bad >> (lane % C::RW) & 1)) {
#pragma unroll
        for (int i = 0; i < C::NC; ++i)
#pragma unroll
            for (int rr = 0; rr < C::QUADS; ++rr)
                out.template quad<D>(C::dim_of(lane, i, rr),
                                     times(make_float4(core.o[i][4 * rr], core.o[i][4 * rr + 1], core.o[i][4 * rr + 2],
                                                       core.o[i][4 * rr + 3]),
                                           inv),
                                     l != 0.0f);
    }
    if (bad) alone(bad, lg);
}

// The four waves' results for the same 16 rows, joined through LDS.
template <typename T, int D, typename F>
__device__ inline void emit_keys(const Args& a, Core<T, D, WAVES_KEYS>& core, const Row& r, int lane, int wave,
                                 int64_t slot, float* smem, F alone) {
    typedef Core<T, D, WAVES_KEYS> C;
    const float l = C::row_sum(core.l);
    __syncthreads();  // every wave is done with its tiles
    float* ml = smem + NW * 16 * D;  // [NW][16] c m, then l
    float* mine = smem + wave * 16 * D;
#pragma unroll
    for (int i = 0; i < C::NC; ++i)
        *reinterpret_cast<floatx4*>(mine + ((i * 4 + lane / 16) * 16 + lane % 16) * 4) = core.o[i];
    if (lane < 16) {
        ml[wave * 16 + lane] = core.m == -INFINITY ? -INFINITY : core.m * a.c - lift<T>;
        ml[64 + wave * 16 + lane] = l;
    }
    __syncthreads();
    float cm = -INFINITY, w[NW], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < NW; ++k) cm = fmaxf(cm, ml[k * 16 + lane % 16]);
#pragma unroll
    for (int k = 0; k < NW; ++k) {
        const float x = ml[k * 16 + lane % 16];
        w[k] = x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(x - cm);
        sum += w[k] * ml[64 + k * 16 + lane % 16];
    }
    const Sink<T> out{a, r.at, r.at / a.x.heads * a.x.ldo + int64_t(r.at % a.x.heads) * D, slot};
    const float lg = log_sum(cm, sum), inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (r.valid && wave == 0 && lane < 16) out.stats(lg);
    float4 v[D / 64];  // quads wave * 4 + lane / 16 + 16 i
    float z = 0.0f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
        v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < NW; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(smem + k * 16 * D + ((wave * 4 + lane / 16 + 16 * i) * 16 + lane % 16) * 4);
            v[i].x += w[k] * x.x, v[i].y += w[k] * x.y, v[i].z += w[k] * x.z, v[i].w += w[k] * x.w;
        }
        z += fmaf(v[i].x, 0.0f, v[i].y * 0.0f) + fmaf(v[i].z, 0.0f, v[i].w * 0.0f);
    }
    uint64_t bad = __ballot(r.valid && sum == sum && !(z == 0.0f));
    bad |= bad >> 32;
    bad = (bad | bad >> 16) & 0xffff;
    if (r.valid && !(bad >> (lane % 16) & 1)) {
#pragma unroll
        for (int i = 0; i < D / 64; ++i) out.template quad<D>(4 * (wave * 4 + lane / 16 + 16 * i), times(v[i], inv), sum != 0.0f);
    }
    if (bad) alone(bad, lg);
}

template <typename T, int D, int TILE, bool MASKED>
__global__ __launch_bounds__(NW * 64, TILE == WAVES_KEYS && D == 512 ? 1 : D == 128 ? 3 : 2) void attention_shared_kernel(Args a) {
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];  // (whole rows: addresses are XORed)
    T* smem = reinterpret_cast<T*>(smem_raw);
    const int tid = int(threadIdx.x), lane = tid % WAVE;
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int G = a.kv.kv_heads, hpg = a.hpg, P = int(a.b.prefix_len), w = a.x.window;
    const int cap = int(a.max_len);

    // The sequence of token `tok`, known to lie in [s0, s1].
    auto seq_in = [&](int64_t tok, int64_t s0, int64_t s1) {
        while (s0 < s1) {
            const int64_t mid = (s0 + s1) / 2;
            if (a.b.start[mid + 1] <= tok)
                s0 = mid + 1;
            else
                s1 = mid;
        }
        return s0;
    };
    auto place = [&](Row& r, int64_t tok, int64_t s0, int64_t s1) {
        r.seq = 0, r.own = 0;
        if (!r.valid) return;
        if (a.b.start) {
            const int64_t s = seq_in(tok, s0, s1);
            r.valid = s < a.b.nseq && tok >= a.b.start[0];
            if (!r.valid) return;
            r.seq = int(s);
            r.own = a.b.lens[s] - int(a.b.start[s + 1] - tok);
        } else {
            r.seq = int(tok);
            r.own = a.b.lens[tok] - 1;
        }
        if constexpr (MASKED) r.own = w > 0 ? __builtin_elementwise_sub_sat(a.tree.positions[tok], P) : 0;
    };
    // The least of the rows' first seen keys (no tile is in use), or `none`.
    auto least = [&](bool valid, int lo, int none) {
        int& first = *reinterpret_cast<int*>(smem_raw);
        __syncthreads();
        if (tid == 0) first = INT_MAX;
        __syncthreads();
        if (valid) atomicMin(&first, lo);
        __syncthreads();
        const int got = first;
        __syncthreads();
        return got == INT_MAX ? none : got / 32 * 32;
    };

    if (int64_t(blockIdx.x) < a.prefix_blocks) {
        typedef Core<T, D, TILE> C;
        constexpr int M = TILE == WAVES_KEYS ? 16 : NW * C::RW;
        // (too few rows for WAVES_16 are never fused)
        const bool fused = TILE != WAVES_KEYS && a.p.fused, whole = TILE != WAVES_KEYS && a.p.whole;
        // Consecutive workgroups go to the 8 XCDs in turn: each XCD takes a
        // run of items, whose tiles share their keys in its L2.
        const int64_t nsplit = whole ? 1 : a.p.np + (fused ? a.p.os : 0);
        const int64_t items = int64_t(a.p.ntile) * G * nsplit;
        const int64_t item = (blockIdx.x % 8) * (a.prefix_blocks / 8) + blockIdx.x / 8;
        if (item >= items) return;
        const int tile = int(item % a.p.ntile);
        const int split = uni(int(item / a.p.ntile % nsplit)), g = uni(int(item / a.p.ntile / nsplit));
        const int64_t rows = a.b.t * hpg, row0 = int64_t(tile) * M;
        const int64_t R = row0 + (TILE == WAVES_KEYS ? 0 : wave * C::RW) + lane % C::RW;
        const int64_t tok = R / hpg;
        const int head = int(g * hpg + R % hpg);
        Row r{R < rows, int(tok * a.x.heads + head), 0, 0};
        const int64_t tok0 = row0 / hpg, tok1 = ((row0 + M < rows ? row0 + M : rows) - 1) / hpg;
        int64_t s0 = tok0, s1 = tok1;
        // The rows' sequences, which prefix keys without a window do not ask
        // for (searches: dependent loads ahead of the first tile).
        auto find = [&] {
            if (a.b.start) {
                s0 = count_le(a.b.start, a.b.nseq, tok0, lane);
                s1 = count_le(a.b.start, a.b.nseq, tok1, lane);
            }
            place(r, r.at / a.x.heads, s0, s1);  // (the row's token again: no register holds it until here)
        };
        const bool placed = w > 0 || whole || split >= a.p.np;
        if (placed)
            find();
        else if (a.b.start)
            r.valid = r.valid && tok >= a.b.start[0] && tok < a.b.start[a.b.nseq];
        C core;
        core.init(r.valid ? static_cast<const T*>(a.x.q) + tok * a.x.ldq + int64_t(head) * D : nullptr, lane);
        const Stream<T, D, TILE> st{a, g, wave, lane, smem};
        [[maybe_unused]] int wb = 0, we = 0;  // MASKED with a window: the split's prefix keys
        if (whole || split < a.p.np) {
            int kb = whole ? 0 : split * a.p.chunk_p, ke = whole ? P : imin(P, kb + a.p.chunk_p);
            const int lo = first_seen(P, r.own, w);
            if (w > 0) {
                // the first key that any of the workgroup's rows sees
                int& first = *reinterpret_cast<int*>(smem_raw);  // (no tile has arrived yet)
                if (tid == 0) first = INT_MAX;
                __syncthreads();
                if (r.valid) atomicMin(&first, lo);
                __syncthreads();
                if constexpr (MASKED) {
                    // (what the tile sees of the prefix is split, not the prefix)
                    const int from = uni(first == INT_MAX ? P : imin(P, first / 32 * 32));
                    const int chunk = whole ? P - from : ((P - from + a.p.np - 1) / a.p.np + 31) / 32 * 32;
                    wb = kb = imin(P, from + (whole ? 0 : split * chunk)), we = ke = imin(P, kb + chunk);
                } else {
                    kb = imax(kb, first == INT_MAX ? ke : first / 32 * 32);
                }
                __syncthreads();
            }
            if (kb < ke) st.run(core, a.b.prefix_table, (P - 1) >> a.page_shift, kb, ke, P, r.valid, lo, P);
        }
        if (fused && (whole || split >= a.p.np)) {
            const int ob = whole ? 0 : (split - a.p.np) * a.p.chunk_o;
            const int oe = whole ? cap : imin(cap, ob + a.p.chunk_o);
            for (int64_t s = s0; s <= s1 && s < a.b.nseq; ++s) {
                // the sequence's tokens of this tile and the keys they see
                const int64_t b0 = a.b.start ? a.b.start[s] : s, b1 = a.b.start ? a.b.start[s + 1] : s + 1;
                const int64_t ta = b0 > tok0 ? b0 : tok0, tb = b1 - 1 < tok1 ? b1 - 1 : tok1;
                if (ta > tb) continue;
                const int len = a.b.lens[s];
                const bool here = r.valid && r.seq == int(s);
                if constexpr (MASKED) {
                    const int base = own_base(a, s), lo = here ? imin(first_seen(0, r.own, w), imax(base, 0)) : 0;
                    const int kb = w > 0 ? imax(ob, least(here, lo, 0)) : ob, ke = imin(oe, len);
                    if (kb < ke)
                        st.template run<true>(core, a.b.table + s * a.b.table_ld, int(a.b.max_pages) - 1, kb, ke,
                                              imin(len, cap), r.valid, lo, here ? imin(len, cap) : 0, base, r.at);
                    continue;
                }
                const int ra = len - int(b1 - ta), rb = len - int(b1 - tb);
                const int kb = imax(ob, first_seen(0, ra, w) / 32 * 32);
                const int ke = imin(oe, rb + 1);
                if (kb >= ke) continue;
                const int lo = here ? first_seen(0, r.own, w) : 0;
                const int hi = here ? imin(r.own + 1, cap) : 0;
                st.run(core, a.b.table + s * a.b.table_ld, int(a.b.max_pages) - 1, kb, ke, imin(len, cap), r.valid, lo,
                       hi);
            }
        }
        Keys in{g, 0, 0, 0, 0};
        if (whole || split < a.p.np)
            in.pb = whole ? 0 : split * a.p.chunk_p, in.pe = whole ? P : imin(P, in.pb + a.p.chunk_p);
        if (MASKED && w > 0) in.pb = wb, in.pe = we;
        if (fused && (whole || split >= a.p.np))
            in.ob = whole ? 0 : (split - a.p.np) * a.p.chunk_o, in.oe = whole ? cap : imin(cap, in.ob + a.p.chunk_o);
        auto alone = [&](uint64_t rows, float lg) {
            if (!placed) find();
            seen_alone<T, D>(a, g, r, rows, lg, lane, split, TILE == WAVES_KEYS ? wave : -1,
                             [&](int i, auto keys) { seen_keys<MASKED>(a, in, r, i, keys); });
        };
        if constexpr (TILE == WAVES_KEYS)
            emit_keys<T, D>(a, core, r, lane, wave, split, reinterpret_cast<float*>(smem_raw), alone);
        else
            emit<T, D, TILE>(a, core, r, lane, split, alone);
        return;
    }

    // Own keys of one sequence: 16 of its rows.
    typedef Core<T, D, WAVES_KEYS> C;
    const int64_t item = int64_t(blockIdx.x) - a.prefix_blocks;
    const int split = uni(int(item % a.p.os)), g = uni(int(item / a.p.os % G));
    const int64_t i = item / a.p.os / G;
    const int per = (hpg + 15) / 16;  // tiles of a single token
    int64_t s, tile, b0, b1;
    if (a.b.start) {
        // Tile i is of the sequence with start[s] hpg / 16 + s <= i: these
        // bounds leave ceil(rows / 16) tiles for every sequence.
        int64_t lo = 0, n = a.b.nseq;
        while (n > 0) {
            const int64_t step = (n + WAVE - 1) / WAVE, k = lo + (lane + 1) * step;
            const int64_t at = k <= lo + n ? k : lo + n;
            const int cnt = __popcll(__ballot(k <= lo + n && int64_t(a.b.start[at]) * hpg / 16 + at <= i));
            const int64_t rest = n - cnt * step;
            lo += cnt * step;
            n = rest < step - 1 ? rest : step - 1;
        }
        s = lo;
        if (s >= a.b.nseq) return;
        b0 = a.b.start[s], b1 = a.b.start[s + 1];
        tile = i - (b0 * hpg / 16 + s);
    } else {
        s = i / per, tile = i % per;
        b0 = s, b1 = s + 1;
    }
    if (tile < 0 || tile * 16 >= (b1 - b0) * hpg) return;
    const int64_t R = tile * 16 + lane % 16;
    const int64_t tok = b0 + R / hpg;
    const int head = int(g * hpg + R % hpg);
    Row r{R < (b1 - b0) * hpg && tok >= 0 && tok < a.b.t, int(tok * a.x.heads + head), int(s), 0};
    const int len = a.b.lens[s];
    r.own = len - int(b1 - tok);
    C core;
    core.init(r.valid ? static_cast<const T*>(a.x.q) + tok * a.x.ldq + int64_t(head) * D : nullptr, lane);
    // the keys that the tile's first and last tokens see
    const int64_t last = (tile * 16 + 15 < (b1 - b0) * hpg ? tile * 16 + 15 : (b1 - b0) * hpg - 1) / hpg;
    const int ra = len - int(b1 - b0 - tile * 16 / hpg), rb = len - int(b1 - b0 - last);
    int kb = imax(split * a.p.chunk_o, first_seen(0, ra, w) / 32 * 32);
    int ke = imin(imin(cap, (split + 1) * a.p.chunk_o), rb + 1);
    const Stream<T, D, WAVES_KEYS> st{a, g, wave, lane, smem};
    if constexpr (MASKED) {
        const int base = own_base(a, s);
        if (r.valid) r.own = w > 0 ? __builtin_elementwise_sub_sat(a.tree.positions[tok], P) : 0;
        const int lo = imin(first_seen(0, r.own, w), imax(base, 0));
        kb = split * a.p.chunk_o, ke = imin(imin(cap, (split + 1) * a.p.chunk_o), len);
        if (w > 0) kb = imax(kb, least(r.valid, lo, 0));
        if (kb < ke)
            st.template run<true>(core, a.b.table + s * a.b.table_ld, int(a.b.max_pages) - 1, kb, ke, imin(len, cap),
                                  r.valid, lo, imin(len, cap), base, r.at);
    } else if (kb < ke) {
        st.run(core, a.b.table + s * a.b.table_ld, int(a.b.max_pages) - 1, kb, ke, imin(len, cap), r.valid,
               first_seen(0, r.own, w), imin(r.own + 1, cap));
    }
    const Keys in{g, 0, 0, split * a.p.chunk_o, imin(cap, (split + 1) * a.p.chunk_o)};
    emit_keys<T, D>(a, core, r, lane, wave, a.p.np + split, reinterpret_cast<float*>(smem_raw), [&](uint64_t rows, float lg) {
        seen_alone<T, D>(a, g, r, rows, lg, lane, a.p.np + split, wave,
                         [&](int i, auto keys) { seen_keys<MASKED>(a, in, r, i, keys); });
    });
}

// out = sum_i w_i O_i / sum_i w_i, w_i = 2^(lg_i - max lg): W waves per
// (token, head), each for every W-th slot, D / 64 values a lane.
template <typename T, int D, int W>
__global__ __launch_bounds__(256) void attention_join_kernel(Args a) {
    constexpr int E = D / WAVE;
    __shared__ float sums[W > 1 ? W : 1][D];
    const int lane = int(threadIdx.x) % WAVE, wave = uni(int(threadIdx.x) / WAVE), mine = wave % W;
    const int64_t rows = a.b.t * a.x.heads;
    const int64_t row = int64_t(blockIdx.x) * (4 / W) + wave / W;
    if (row >= rows) return;
    const int64_t tok = row / a.x.heads, head = row - tok * a.x.heads;
    if (token_row(a.b, tok, lane).seq < 0) return;  // (W > 1: the whole workgroup)
    const int slots = int(a.p.slots());
    float lg[2], w[2];  // the lane's slots (at most 64 of each kind)
#pragma unroll
    for (int j = 0; j < 2; ++j)
        lg[j] = lane + j * WAVE < slots ? a.part_lg[(lane + j * WAVE) * rows + row] : -INFINITY;
    const float most = wave_max(fmaxf(lg[0], lg[1]));
#pragma unroll
    for (int j = 0; j < 2; ++j) w[j] = lg[j] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(lg[j] - most);
    const float l = wave_sum(w[0] + w[1]), inv = l == 0.0f ? 0.0f : 1.0f / l;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.0f;
    for (int i0 = 0; i0 < slots; i0 += WAVE) {
        const float wl = (i0 ? w[1] : w[0]) * inv;
        const int n = slots - i0 < WAVE ? slots - i0 : WAVE;
        // (eight slots' loads under way; what a slot without a share holds
        // was not written)
#pragma unroll 1
        for (int i = mine; i < n; i += 8 * W) {
            float x[8][E];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int at = i + k * W < n ? i + k * W : 0;
                const float* o = a.part_o + (int64_t(i0 + at) * rows + row) * D + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) x[k][e] = o[e];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float f = i + k * W < n ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wl), i + k * W)) : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] += f == 0.0f ? 0.0f : f * x[k][e];
            }
        }
    }
    if constexpr (W > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) sums[wave][lane * E + e] = v[e];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            v[e] = 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) v[e] += sums[k][lane * E + e];
        }
    }
    T* out = static_cast<T*>(a.x.out) + tok * a.x.ldo + head * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = mean<T>(v[e]);
    if (lane == 0 && a.x.lse) a.x.lse[row] = log_sum(most, l) * 0.69314718055994531f;
}

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

// Work items fill the places that the chip's 256 CUs are counted to have
// where the keys are long enough to be split.  (The window is no part of it.)
[[maybe_unused]] Plan plan(const PagedKv& kv, const PagedBatch& b, int heads) {
    Plan p{};
    const int64_t hpg = heads / kv.kv_heads, rows = b.t * hpg, max_len = b.max_pages * kv.page, P = b.prefix_len;
    p.fused = rows >= 32 * b.nseq;
    if (!p.fused && rows <= 16)
        p.tile = WAVES_KEYS;
    else if (rows <= 64 || kv.head_dim == 512)
        p.tile = WAVES_16;
    else
        p.tile = WAVES_32;
    const int64_t M = p.tile == WAVES_KEYS ? 16 : p.tile == WAVES_16 ? 64 : 128;
    p.ntile = int((rows + M - 1) / M);
    const int64_t base = p.ntile * int64_t(kv.kv_heads);
    // Two workgroups on each of 256 CUs (head_dim 64: four) take up the launch
    // at once; a few items more wait for a second round (504 items of 512-wide
    // heads 57 us, 567 78 us).  Launches of 512-wide heads with own items hold
    // one a CU, by LDS, and are counted alike.
    const int64_t SLOTS = kv.head_dim == 64 ? 1024 : 512;
    auto splits = [&](int64_t keys, int64_t k, int64_t least, int& n, int& chunk) {
        k = std::max<int64_t>(1, std::min<int64_t>({k, (keys + least - 1) / least, 64}));
        chunk = int(up((keys + k - 1) / k, 32));
        n = int((keys + chunk - 1) / chunk);
    };
    p.os = 1, p.chunk_o = int(std::min<int64_t>(up(max_len, 32), INT_MAX / 2));
    if (p.fused) {
        p.whole = base * 2 >= SLOTS;
        if (!p.whole) {
            const int64_t all = SLOTS / base;  // shared out by the keys' numbers
            const int64_t own = std::max<int64_t>(1, all * max_len / (P + max_len));
            splits(max_len, P > 0 ? own : all, 128, p.os, p.chunk_o);
            if (P > 0) splits(P, all - p.os, 128, p.np, p.chunk_p);
        }
        return p;
    }
    // A prefix split writes and reads 8 bytes a row and head dim, and reads
    // 4 a key of its own: beyond 2 keys for 3 rows splits cost more than
    // they fill (208 x 2 rows on 8,000 keys: 12 / 16 / 20 / 32 splits 45 / 43
    // / 46 / 55 us), unless CUs stay empty.
    if (P > 0) splits(P, std::min(SLOTS / base, std::max(SLOTS / 2 / base, 2 * P / (3 * rows))), 64, p.np, p.chunk_p);
    const int64_t per = (hpg + 15) / 16;
    p.own_tiles = b.start ? rows / 16 + b.nseq : b.nseq * per;
    splits(max_len, SLOTS / (p.own_tiles * kv.kv_heads), 128, p.os, p.chunk_o);
    return p;
}

void check(const PagedKv& kv, const PagedBatch& b, int heads, const char* who) {
    const std::string w(who);
    check_kv(kv, who);
    check_batch(b, kv, who);
    if (heads <= 0 || heads > 4096 || heads % kv.kv_heads)
        fail(E_INVALID, w + ": heads must be a multiple of kv_heads, at most 4096");
    if (b.t * heads >= (1 << 26)) fail(E_INVALID, w + ": t * heads must stay below 2^26");
}

void check_rows(const PagedKv& kv, const SharedAttn& x, const char* who) {
    const std::string w(who);
    const int64_t width = int64_t(x.heads) * kv.head_dim;
    if (!x.q || !x.out || !aligned16(x.q) || !aligned16(x.out))
        fail(E_INVALID, w + ": q and out must be 16-byte aligned device pointers");
    if (x.ldq < width || x.ldq % 8 || x.ldo < width || x.ldo % 8)
        fail(E_INVALID, w + ": ldq and ldo must hold the heads and be multiples of 8");
    if (!(x.scale > 0.0f) || x.scale > 1e30f) fail(E_INVALID, w + ": scale must be positive and finite");
    if (x.window < 0) fail(E_INVALID, w + ": window must not be negative");
}

[[maybe_unused]] int64_t part_bytes(const Plan& p, const PagedKv& kv, const PagedBatch& b, int heads) {
    const int64_t n = p.slots();
    return n <= 1 ? 0 : n * b.t * heads * (kv.head_dim * 4 + 4);
}

template <typename T, int D, bool MASKED>
void launch_d(hipStream_t s, const Args& a, unsigned blocks) {
    // tiles: 2 buffers of 32 keys (head_dim 512: 16), or 4 waves x 16 keys,
    // of K and V; the waves' join: 4 x 16 rows of f32 and their
    // statistics
    constexpr unsigned lds_rows = 2 * (D == 512 ? 16 : 32) * D * 4;
    constexpr unsigned lds_keys = NW * 16 * D * 4 + 2 * NW * 16 * 4;
    const unsigned lds = a.p.fused ? lds_rows : std::max(lds_keys, lds_rows);
    static std::atomic<uint64_t> lds_set[3];  // by tile: the devices, once per instantiation
    int device = 0;
    OMG_HIP(hipGetDevice(&device));
    auto go = [&](auto kernel) {
        const uint64_t bit = uint64_t(1) << (device & 63);
        if (device > 63 || !(lds_set[a.p.tile].load(std::memory_order_relaxed) & bit)) {
            OMG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, int(std::max(lds_keys, lds_rows))));
            lds_set[a.p.tile].fetch_or(bit, std::memory_order_relaxed);
        }
        kernel<<<dim3(blocks), dim3(NW * 64), lds, s>>>(a);
    };
    auto joined = [&] {
        OMG_HIP(hipGetLastError());
        if (!a.part_o) return;
        const int64_t rows = a.b.t * a.x.heads;
        if (a.p.slots() > 8)
            attention_join_kernel<T, D, 4><<<dim3(unsigned(rows)), dim3(256), 0, s>>>(a);
        else
            attention_join_kernel<T, D, 1><<<dim3(unsigned((rows + 3) / 4)), dim3(256), 0, s>>>(a);
        OMG_HIP(hipGetLastError());
    };
    if (a.p.tile == WAVES_KEYS)
        go(attention_shared_kernel<T, D, WAVES_KEYS, MASKED>);
    else if (a.p.tile == WAVES_16)
        go(attention_shared_kernel<T, D, WAVES_16, MASKED>);
    else if constexpr (D < 512) {
        go(attention_shared_kernel<T, D, WAVES_32, MASKED>);
    }
    joined();
}

template <typename T, bool MASKED>
void launch_t(hipStream_t s, const Args& a, unsigned blocks) {
    switch (a.kv.head_dim) {
        case 64: return launch_d<T, 64, MASKED>(s, a, blocks);
        case 128: return launch_d<T, 128, MASKED>(s, a, blocks);
        case 256: return launch_d<T, 256, MASKED>(s, a, blocks);
        default: return launch_d<T, 512, MASKED>(s, a, blocks);
    }
}

template <bool MASKED, typename F>
void launch_attention(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const SharedAttn& x, const TreeMask& tree,
                      F planned, void* workspace, size_t bytes, const char* who) {
    const std::string name(who);
    check(kv, b, x.heads, who);
    check_rows(kv, x, who);
    Args a{};
    a.kv = kv, a.b = b, a.x = x, a.tree = tree;
    a.p = planned(kv, b, x.heads);
    a.hpg = x.heads / kv.kv_heads;
    a.page_shift = log2_of(kv.page);
    a.max_len = b.max_pages * kv.page;
    a.c = x.scale * 1.4426950408889634f;
    const int64_t need = part_bytes(a.p, kv, b, x.heads);
    if (int64_t(bytes) < need) fail(E_CAPACITY, name + ": the workspace needs " + std::to_string(need) + " bytes");
    if (need) {
        if (!workspace || !aligned16(workspace)) fail(E_INVALID, name + ": the workspace must be 16-byte aligned");
        a.part_o = static_cast<float*>(workspace);
        a.part_lg = a.part_o + a.p.slots() * b.t * x.heads * kv.head_dim;
    }
    const int64_t nsplit = a.p.whole ? 1 : a.p.np + (a.p.fused ? a.p.os : 0);
    a.prefix_blocks = up(int64_t(a.p.ntile) * kv.kv_heads * nsplit, 8);
    const int64_t blocks = a.prefix_blocks + (a.p.fused ? 0 : a.p.own_tiles * kv.kv_heads * a.p.os);
    if (blocks >= MAX_BLOCKS) fail(E_CAPACITY, name + ": too many work items");
    kv.dtype == ELEM_F16 ? launch_t<half_t, MASKED>(s, a, unsigned(blocks)) : launch_t<bf16_t, MASKED>(s, a, unsigned(blocks));
}

}  // namespace

}  // namespace omg
