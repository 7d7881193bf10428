// The attention weight that each cached row gathers:
//   weights[s][g][i] += sum of exp(scale q . k_i - lse) over the sequence's
// tokens that see its row i and the query heads of KV head g, lse the log sums
// that attention left.  No softmax runs here, so every key's sum stands alone:
// what a row holds reaches its own weight and no other.
//
// Keys stay, queries pass by.  A wave holds its keys in registers, as the A
// operand straight from their pages, and S = K Q^T leaves a key's scores in
// the same registers whatever query tile comes: probabilities add up there, and
// the lanes (queries) are summed once at the end, in an order that the sizes
// fix.  A weight is read and written by one lane of one wave.
//
// Few rows a sequence (steps of decoding): weights_few_kernel, 16 keys x 16
// rows, bound by reading K.  Many (prompts): weights_many_kernel, a wave 64 keys
// (512-wide heads: 32), query tiles of 32 rows in LDS for its four waves; where
// keys are few the queries are split and the parts' sums added by
// weights_join_kernel.
//
// Measured, and what bounds it:
//   64 sequences of 6,100 rows x 8 KV heads of 128 (bf16), one token each: 170 us,
//     4.9 TB/s: the keys' bytes.
//   12 sequences of 2,000 rows x 1 KV head of 256 (f16): 5.8 us: latency.
//   a prompt of 8,000 tokens x 8 heads of 256 on 4 KV heads (f16): 148 us
//     and the join's 5 alone, 141 a call in a row, 930 TFLOP/s of the 1,154 that a
//     product of 8,192^3 reaches: MFMAs 48 % and vector instructions 53 % of the busy
//     SIMDs' cycles.  On random data the chip lowers its clock, for 16 x 16 x 32
//     products less than for 32 x 32 x 16 (from registers alone 1,990 and 1,660
//     TFLOP/s, on zeros both 2,470): 174 -> 165 us when it was that, at 128-wide
//     heads 160 -> 132.
#include <algorithm>
#include <atomic>
#include <climits>
#include <string>

#include "common.h"
#include "kern_common.h"
#include "paged.h"

namespace omg {

namespace {

typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ inline floatx4 mfma16(half8 a, half8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ inline floatx4 mfma16(bf16x8 a, bf16x8 b, floatx4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

struct Args {
    PagedKv kv;
    PagedBatch b;
    AttnWeights x;
    int hpg, page_shift;
    int64_t max_len;
    int64_t blocks;  // few: key chunks, many: key blocks of a sequence
    int chunk;       // few: keys of a workgroup
    int splits;      // many: of a sequence's tokens
    float* part;     // [splits][nseq * kv_heads][max_len], null: into the weights
};

// A sequence's tokens, its rows in the cache and the row of its first token.
struct Seq {
    int tok, n, len, base;
};
__device__ inline Seq sequence(const Args& a, int64_t s) {
    const int tok = a.b.start ? a.b.start[s] : int(s), n = a.b.start ? a.b.start[s + 1] - tok : 1;
    const int len = a.b.lens[s] < 0 ? 0 : a.b.lens[s];
    return {tok, n, len < a.max_len ? len : int(a.max_len), len - n};
}

// exp(s scale - lse); lse of minus infinity (a token that sees nothing) leaves 0.
__device__ inline float prob(float s, float scale, float neg_lse) {
    return __builtin_amdgcn_exp2f(fmaf(s, scale, neg_lse) * 1.4426950408889634f);
}
__device__ inline float negated(float lse) { return lse == -INFINITY ? -INFINITY : -lse; }

__device__ inline float sum16(float v) {  // over the 16 lanes of a row, the same bits in each
    v += dpp_f32<0xb1>(v);
    v += dpp_f32<0x4e>(v);
    v += dpp_f32<0x141>(v);
    v += dpp_f32<0x140>(v);
    return v;
}

// The elements of a row's page (null: not in the pool).
template <typename T>
__device__ inline const T* key_row(const Args& a, const int32_t* table, int row, int g, int D) {
    const int i = row >> a.page_shift;
    if (i >= a.b.max_pages) return nullptr;
    const int64_t p = table[i];
    if (p < 0 || p >= a.kv.npages) return nullptr;
    return static_cast<const T*>(a.kv.k) + p * a.kv.page_stride + (int64_t(g) * a.kv.page + (row & (a.kv.page - 1))) * D;
}

// Four waves, each every fourth group of U 16-key tiles of the chunk.  (More
// waves on a CU keep more loads under way than more tiles in a wave: 128-wide
// heads with four tiles, 130 registers, 200 us, with one, 58, 170.)
template <typename T, int D>
__global__ __launch_bounds__(256) void weights_few_kernel(Args a) {
    typedef typename Vec8<T>::type frag;
    constexpr int NS = D / 32, U = D >= 128 ? 1 : 2, KEYS = 16 * U;
    const int lane = int(threadIdx.x) % WAVE, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    const int64_t id = blockIdx.x, list = id / a.blocks, s = list / a.kv.kv_heads;
    const int g = int(list - s * a.kv.kv_heads), from = int(id - list * a.blocks) * a.chunk;
    const Seq q = sequence(a, s);
    const int to = from + a.chunk < q.len ? from + a.chunk : q.len;
    if (from >= to || q.n <= 0) return;
    const int32_t* table = a.b.table + s * a.b.table_ld;
    float* out = a.x.weights + list * a.x.ldw;
    const int rows = q.n * a.hpg, w = a.x.window;
    // keys that a window hides from the first token are seen by none
    const int lo = w > 0 && q.base + 1 > w ? q.base + 1 - w : 0;

    frag qf[NS];
    float nl = -INFINITY;  // the row's negated lse
    int own = 0;           // the row's token's row in the cache
    auto load = [&](int r0) {
        const int r = r0 + lane % 16, tok = r / a.hpg, head = g * a.hpg + r - tok * a.hpg;
        const int64_t at = q.tok + tok;
        const bool valid = r < rows && at >= 0 && at < a.b.t;
        nl = valid ? negated(a.x.lse[at * a.x.heads + head]) : -INFINITY;
        own = valid ? q.base + tok : -1;
        const T* p = static_cast<const T*>(a.x.q) + (valid ? at * a.x.ldq + int64_t(head) * D : 0) + 8 * (lane / 16);
        frag z{};
#pragma unroll
        for (int st = 0; st < NS; ++st) qf[st] = valid ? *reinterpret_cast<const frag*>(p + 32 * st) : z;
    };
    load(0);
    for (int k0 = from + wave * KEYS; k0 < to; k0 += 4 * KEYS) {
        if (k0 + KEYS <= lo) continue;
        frag kf[U][NS];
        bool there[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (a tile lies in one page, which is whole in the pool)
            const T* p = k0 + 16 * u < to ? key_row<T>(a, table, k0 + 16 * u, g, D) : nullptr;
            there[u] = p != nullptr;
            if (!p) continue;
            p += int64_t(lane % 16) * D + 8 * (lane / 16);
#pragma unroll
            for (int st = 0; st < NS; ++st) kf[u][st] = *reinterpret_cast<const frag*>(p + 32 * st);
        }
        float sum[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[u][r] = 0.0f;
        for (int r0 = 0; r0 < rows; r0 += 16) {
            if (rows > 16) load(r0);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (!there[u]) continue;
                floatx4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < NS; ++st) sc = mfma16(kf[u][st], qf[st], sc);
                const int first = k0 + 16 * u + 4 * (lane / 16);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool see = first + r <= own && (w == 0 || own - (first + r) < w) && nl != -INFINITY;
                    const float p = prob(sc[r], a.x.scale, nl);
                    sum[u][r] += see ? p : 0.0f;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[u][r] = sum16(sum[u][r]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int key = k0 + 16 * u + 4 * (lane / 16) + lane % 16;
            float mine = sum[u][0];
#pragma unroll
            for (int r = 1; r < 4; ++r) mine = lane % 16 == r ? sum[u][r] : mine;
            if (there[u] && lane % 16 < 4 && key < to) out[key] += mine;
        }
    }
}

// Many rows.
template <typename T, int D>
struct Many {
    static constexpr int NB = D >= 512 ? 2 : 4;  // 16-key blocks of a wave
    static constexpr int KEYS = 4 * 16 * NB;     // of a workgroup
    static constexpr int CH = D / 8, RPI = 512 / D > 0 ? 512 / D : 1;
    static constexpr int INS = 32 * D * 2 / 1024 / 4;  // 1 KiB pieces of a query tile per wave
    static constexpr int TILE = 32 * D;
    static constexpr int BUFS = D >= 512 ? 2 : 4;  // query tiles in LDS
    static __device__ int swz(int row) { return CH >= 16 ? row & 15 : row >> 1 & 7; }
};

// N pieces of 1 KiB to LDS from the lanes' offsets behind `base`; zeros from
// `bytes` on.
template <int N>
__device__ inline void to_lds(const char* base, int bytes, const uint32_t* off, void* dst) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < N; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(static_cast<char*>(dst) + 1024 * i), 16, off[i], 0, 0, 0);
}

// A value a lane.  (Not by a global load to LDS: behind one the compiler waits
// for all LDS reads where it needs the oldest.)
__device__ inline void log_sums_to_lds(const char* base, int bytes, uint32_t off, void* dst) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), (short)0, bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)dst, 4, off, 0, 0, 0);
}

// All but the last N loads have arrived, and LDS reads.
template <int N>
__device__ inline void wait_loads() {
    static_assert(N < 64, "vmcnt holds 6 bits");
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// A work item: the key block of KEYS rows from kb on of a list, and the tokens [ta, tb) of
// the sequence's, its split's of those that see a key of the block.
struct Item {
    int g, kb, split, ta, tb;
    int64_t s, list;
    Seq q;
};
template <int KEYS>
__device__ inline Item item(const Args& a, int64_t id) {
    Item x;
    // KV heads fastest: the workgroups of one XCD share a few heads' queries.  Blocks
    // slowest: the longest items first, and a place's items in a row are not one
    // sequence's (30 x 300 tokens x 32 heads of 128 53 -> 43 us, 114 x 382 x 8 of 256
    // 97 -> 75).  A last split is short: not always the same XCD's.
    const int G = a.kv.kv_heads;
    x.g = int(id % G);
    id /= G;
    const int turn = int(id % a.splits);
    id /= a.splits;
    x.kb = int(id / a.b.nseq) * KEYS, x.split = int((turn + id) % a.splits);
    x.s = id % a.b.nseq, x.list = x.s * G + x.g;
    x.q = sequence(a, x.s);
    const int w = a.x.window, tile = 32 / (a.hpg < 32 ? a.hpg : 32);  // whole query tiles
    int from = x.kb > x.q.base ? x.kb - x.q.base : 0, until = x.q.n;
    // (token rows outside the batch's are nobody's)
    if (x.q.tok < 0 && from < -x.q.tok) from = -x.q.tok;
    if (until > a.b.t - x.q.tok) until = int(a.b.t - x.q.tok);
    if (w > 0) {
        const int64_t end = int64_t(x.kb) + KEYS - 1 + w - x.q.base;  // own < key + w
        if (until > end) until = int(end < 0 ? 0 : end);
    }
    const int per = until > from ? (until - from + a.splits * tile - 1) / (a.splits * tile) * tile : 0;
    x.ta = from + x.split * per, x.tb = x.ta + per < until ? x.ta + per : until;
    return x;
}

// What a key gathers in a work item, with a row a lane and no row that does not see it:
// until the sum is NaN.
template <typename T, int D>
__device__ inline float key_alone(int key, int lane) {
    // (the item from the launch's arguments again: no register holds any of it until
    // here; with them held, 8,000 tokens at a window of 512 took 56 us for 53)
    uint64_t args = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
    int id = int(blockIdx.x);
    asm volatile("" : "+s"(args), "+s"(id));
    const Args& a = *reinterpret_cast<const Args*>(args);
    const Item it = item<Many<T, D>::KEYS>(a, id);
    const T* k = key_row<T>(a, a.b.table + it.s * a.b.table_ld, key, it.g, D);
    if (!k) return 0.0f;
    float sum = 0.0f;
#pragma unroll 1
    for (int64_t r0 = int64_t(it.ta) * a.hpg, end = int64_t(it.tb) * a.hpg; r0 < end; r0 += WAVE) {
        const int64_t r = r0 + lane, tok = r / a.hpg, own = it.q.base + tok, at = it.q.tok + tok;
        const int head = it.g * a.hpg + int(r - tok * a.hpg);
        const bool see = r < end && key <= own && (a.x.window == 0 || own - key < a.x.window);
        const float nl = see ? negated(a.x.lse[at * a.x.heads + head]) : -INFINITY;
        if (nl != -INFINITY) {
            const T* x = static_cast<const T*>(a.x.q) + at * a.x.ldq + int64_t(head) * D;
            float s = 0.0f;
#pragma unroll 4
            for (int c = 0; c < D; c += 8) {
                float u[8], v[8];
                load8(x + c, u), load8(k + c, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = fmaf(u[i], v[i], s);
            }
            sum += prob(s, a.x.scale, nl);
        }
        if (__any(sum != sum)) break;
    }
    return wave_sum(sum);
}

template <typename T, int D>
__global__ __launch_bounds__(256, 2) void weights_many_kernel(Args a) {
    typedef typename Vec8<T>::type frag;
    typedef Many<T, D> M;
    constexpr int NB = M::NB, NS = D / 32, E = 4 * NB;  // blocks; steps of a product; scores of a lane
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
    T* smem = reinterpret_cast<T*>(smem_raw);  // BUFS query tiles
    float* log_sums = reinterpret_cast<float*>(smem_raw + M::BUFS * M::TILE * 2);  // [BUFS][4][64]
    const int lane = int(threadIdx.x) % WAVE, wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / WAVE);
    const Item it = item<M::KEYS>(a, blockIdx.x);
    const Seq q = it.q;
    if (it.kb >= q.len) return;
    const int g = it.g, hpg = a.hpg, kb = it.kb, k0 = kb + wave * 16 * NB, w = a.x.window, ta = it.ta, tb = it.tb;
    // Query tiles of the heads of TPT tokens or 32 heads of one, so that a lane's row
    // is the same token and head past the tile's first in each.
    const int heads = hpg < 32 ? hpg : 32, TPT = 32 / heads, parts = (hpg + 31) / 32;
    float sum[E];  // of key 16 (e / 4) + 4 (lane / 16) + e % 4 of the wave's
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    const int32_t* table = a.b.table + it.s * a.b.table_ld;
    if (ta < tb) {
        frag kf[NB][NS];
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int row = k0 + 16 * j + lane % 16;
            const T* p = row < q.len ? key_row<T>(a, table, row, g, D) : nullptr;
            frag z{};
#pragma unroll
            for (int st = 0; st < NS; ++st)
                kf[j][st] = p ? *reinterpret_cast<const frag*>(p + 32 * st + 8 * (lane / 16)) : z;
        }
        const int have = tb - ta, ntile = (have + TPT - 1) / TPT * parts;
        const int64_t tok0 = q.tok + ta;
        const char* qb = reinterpret_cast<const char*>(static_cast<const T*>(a.x.q) + tok0 * a.x.ldq + int64_t(g) * hpg * D);
        uint32_t off[M::INS];  // of the rows that the lane loads a chunk of; no row: past all
#pragma unroll
        for (int i = 0; i < M::INS; ++i) {
            const int r = (wave * M::INS + i) * M::RPI + lane / M::CH, t = r / heads;
            off[i] = (t < TPT ? uint32_t(t * a.x.ldq + (r - t * heads) * D) * 2 : 1u << 31) + ((lane % M::CH) ^ M::swz(r)) * 16;
        }
        const int mt = lane % 32 / heads, mh = lane % 32 - mt * heads;  // of the row whose log sum it loads
        int t0 = 0, part = 0;                                           // of the next tile
        const float* lse = a.x.lse + tok0 * a.x.heads + g * hpg;
        const uint32_t lse_off = uint32_t(mt * a.x.heads + mh) * 4;
        // Rows that are not there arrive as zeros, or as others, and have a
        // negated log sum of minus infinity.  (A load each way: the waits count.)
        auto issue = [&](T* dst) {
            const int64_t skip = t0 * a.x.ldq + part * 32 * D;
            const int64_t left = t0 < have ? 2 * ((have - 1) * a.x.ldq + hpg * D - skip) : 0;
            to_lds<M::INS>(qb + (t0 < have ? 2 * skip : 0), int(left < INT_MAX ? left : INT_MAX), off, dst + wave * M::INS * 512);
            // (log sums into registers would be waited for, and all loads before them, tile by tile)
            const int64_t past = int64_t(t0) * a.x.heads + part * 32, rest = t0 < have ? 4 * (int64_t(have) * a.x.heads - g * hpg - past) : 0;
            log_sums_to_lds(reinterpret_cast<const char*>(lse + (t0 < have ? past : 0)), int(rest < INT_MAX ? rest : INT_MAX),
                            lse_off, log_sums + (int(dst - smem) / M::TILE * 4 + wave) * WAVE);
            if (++part == parts) part = 0, t0 += TPT;
        };
        // BUFS - 1 tiles are under way; behind the last one the loads go on, to
        // nothing, so that a wait leaves the same number out.
        constexpr int AHEAD = M::BUFS - 1;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) issue(smem + i * M::TILE);
        // The lane's query rows are lane % 16 of the tile's two halves.
        const int ht[2] = {lane % 16 / heads, (16 + lane % 16) / heads};
        const int hh[2] = {lane % 16 - ht[0] * heads, 16 + lane % 16 - ht[1] * heads};
        const uint32_t my_row = uint32_t(lane % 16 * D * 2 + ((lane / 16) ^ M::swz(lane % 16)) * 16);
        typedef __attribute__((address_space(3))) frag* operand;
        int at = 0, tok = 0, hp = 0;  // of the tile at hand: its buffer, first token and part
        // The next tile has landed: the LDS address of the lane's first row, and
        // the rows' negated log sums.
        auto arrive = [&](float* nl) {
            wait_loads<(AHEAD - 1) * (M::INS + 1)>();
            __syncthreads();
            issue(smem + (at + AHEAD) % M::BUFS * M::TILE);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float lse = log_sums[(at * 4 + wave) * WAVE + 16 * h + lane % 16];
                nl[h] = tok + ht[h] < have && ht[h] < TPT && hp * 32 + hh[h] < hpg ? negated(lse) : -INFINITY;
            }
            uint32_t row = uint32_t(uintptr_t((lds_ptr)(smem + at * M::TILE))) + my_row;
            asm volatile("" : "+v"(row));  // (or all steps' addresses are kept in registers)
            at = (at + 1) % M::BUFS;
            return row;
        };
        // The operand of step n of a tile: of rows 16 (n / NS), dims 32 (n % NS).
        auto read = [&](uint32_t row, int n) {
            return *(operand)(uintptr_t)((row ^ uint32_t(64 * (n % NS))) + uint32_t(n / NS * 16 * D * 2));
        };
        auto next = [&] {
            if (++hp == parts) hp = 0, tok += TPT;
        };
        // Tiles [f0, f1) hold tokens that see all keys of the block.
        int f0 = q.base + ta >= kb + M::KEYS - 1 ? 0 : (kb + M::KEYS - 1 - q.base - ta + TPT - 1) / TPT * parts, f1 = ntile;
        if (w > 0) {
            const int64_t most = int64_t(w) + kb - q.base - ta - TPT;  // the last first token
            f1 = most < 0 ? 0 : int(most / TPT + 1 < f1 ? (most / TPT + 1) * parts : f1);
        }
        if (hpg > 32 && hpg % 32) f0 = ntile;  // (a part's last rows are other heads')
        f0 = f0 < ntile ? f0 : ntile, f1 = f1 < ntile ? f1 : ntile, f1 = f1 > f0 ? f1 : f0;
#pragma unroll 1
        for (int i = 0; i < ntile;) {
            if (i != f0 || f0 == f1) {
                // Tiles at the diagonal and the window's end.
                const int end = i < f0 ? f0 : ntile;
#pragma unroll 1
                for (; i < end; ++i, next()) {
                    float nl[2];
                    const uint32_t row = arrive(nl);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        floatx4 sc[NB];
#pragma unroll
                        for (int j = 0; j < NB; ++j) sc[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int st = 0; st < NS; ++st) {
                            const frag qf = read(row, h * NS + st);
#pragma unroll
                            for (int j = 0; j < NB; ++j) sc[j] = mfma16(kf[j][st], qf, sc[j]);
                        }
                        // (the lane's keys past k0 + 4 (lane / 16): constants of an element)
                        const int last = q.base + ta + tok + ht[h] - k0 - 4 * (lane / 16);
                        const int from = w == 0 ? INT_MIN : __builtin_elementwise_sub_sat(last, w);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const int key = 16 * (e / 4) + e % 4;
                            const float p = prob(sc[e / 4][e % 4], a.x.scale, nl[h]);
                            sum[e] += key <= last && key > from && nl[h] != -INFINITY ? p : 0.0f;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                continue;
            }
            // The scores of half a tile wait for the next half's MFMAs, in whose
            // shadow their exponentials run.  A step: the MFMAs of one operand, the
            // operand of the step READ on and a part of the half before, in this
            // order.  (Left alone, the compiler reads one operand and waits for it.)
            // From the third step on: the last half's MFMAs are still under way.
            constexpr int LATE = NS > 2 ? 2 : 1, READ = 4;
            auto first = [](int st) { return st < LATE ? 0 : (st - LATE) * E / (NS - LATE); };
            floatx4 was[NB];
            float was_nl = -INFINITY;
#pragma unroll
            for (int j = 0; j < NB; ++j) was[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (; i < f1; ++i, next()) {
                float nl[2];
                const uint32_t row = arrive(nl);
                frag qf[READ];
#pragma unroll
                for (int k = 0; k < READ; ++k) qf[k] = read(row, k);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    floatx4 sc[NB];
#pragma unroll
                    for (int j = 0; j < NB; ++j) sc[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int st = 0; st < NS; ++st) {
                        const int n = h * NS + st;
#pragma unroll
                        for (int j = 0; j < NB; ++j) sc[j] = mfma16(kf[j][st], qf[n % READ], sc[j]);
                        if (n + READ < 2 * NS) qf[n % READ] = read(row, n + READ);
#pragma unroll
                        for (int e = first(st); e < first(st + 1); ++e) sum[e] += prob(was[e / 4][e % 4], a.x.scale, was_nl);
                        __builtin_amdgcn_sched_barrier(0);
                    }
#pragma unroll
                    for (int j = 0; j < NB; ++j) was[j] = sc[j];
                    was_nl = nl[h];
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += prob(was[e / 4][e % 4], a.x.scale, was_nl);
        }
        wait_loads<0>();  // (no load may find the LDS another workgroup's)
    }
    // Lane 16 g + e has the sum of element e of the group.
    float mine = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float v = sum16(sum[e]);
        mine = lane % 16 == e ? v : mine;
    }
    const int e = lane % 16, key = k0 + 16 * (e / 4) + 4 * (lane / 16) + e % 4;
    // Tiles that see the whole block add up all their rows: a zero for one that no token
    // has or whose token sees nothing, but NaN where its score is infinite or NaN (an
    // infinite key's with a row of zeros is).  So a key whose sum is NaN is taken again:
    // 4,096 tokens x 7 heads of 256 with one such key in 1,000 98 us for 69, with nothing
    // else 5.0 ms, where they are NaN themselves 1.3 ms.  (A choice for each probability
    // instead takes 2 % of 256-wide, 3 % of 128-wide and 7 % of 64-wide heads' time, always.)
    for (uint64_t again = __ballot(e < E && key < q.len && mine != mine); again; again &= again - 1) {
        const int from = __builtin_ctzll(again);
        const float v = key_alone<T, D>(__builtin_amdgcn_readlane(key, from), lane);
        mine = lane == from ? v : mine;
    }
    if (e >= E || key >= q.len || !key_row<T>(a, table, key, g, D)) return;
    if (a.part)
        a.part[(it.split * a.b.nseq * a.kv.kv_heads + it.list) * a.max_len + key] = mine;
    else
        a.x.weights[it.list * a.x.ldw + key] += mine;
}

// The splits' sums, in their order.
__global__ __launch_bounds__(256) void weights_join_kernel(Args a) {
    const int64_t list = blockIdx.y, s = list / a.kv.kv_heads, key = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const Seq q = sequence(a, s);
    if (key >= q.len) return;
    const int64_t p = a.b.table[s * a.b.table_ld + (key >> a.page_shift)];
    if (p < 0 || p >= a.kv.npages) return;
    float v = 0.0f;
#pragma unroll 8
    for (int i = 0; i < a.splits; ++i) v += a.part[(i * a.b.nseq * a.kv.kv_heads + list) * a.max_len + key];
    a.x.weights[list * a.x.ldw + key] += v;
}

void check(const PagedKv& kv, const PagedBatch& b, int heads) {
    check_kv(kv, "attention_weights");
    check_batch(b, kv, "attention_weights");
    if (heads <= 0 || heads > 4096 || heads % kv.kv_heads)
        fail(E_INVALID, "attention_weights: heads must be a multiple of kv_heads, at most 4096");
    if (b.t * heads >= (1 << 26)) fail(E_INVALID, "attention_weights: t * heads must stay below 2^26");
}

// Few rows a sequence, in the mean: lengths lie on the device.  (A prompt among many
// single tokens goes with these: 8,000 tokens and 300 single ones x 12 heads of 64 9.0 ms,
// in a call each 0.12 and 0.18.)
bool few(const PagedKv& kv, const PagedBatch& b, int heads) { return b.t * (heads / kv.kv_heads) <= 32 * b.nseq; }

int many_keys(int head_dim) { return head_dim == 512 ? 128 : 256; }

// The splits of a key block's queries of least time: the longest item's tiles,
// four more for its start and end, or all items' over the places that the chip
// has and a quarter of one at the launch's end; for sequences of the mean number of
// tokens, and of several three quarters of the items, since most are shorter than
// the table.  (A split takes its part of the tokens that see the block, so that late
// blocks' items, which come last, are short: of all tokens, 4,096 x 32 heads of 128
// 127 us for 100, 8,000 x 8 of 256 on 4 KV heads 161 for 145.  Those 8,000: 4 / 6 / 10
// / 16 / 32 splits 174 / 144 / 146 / 147 / 169, 10 is what this gives; 600 x 8 of 512 on
// one: 8 / 16 / 48 37 / 25 / 18; 9 x 200 x 15 of 64 on 5: 1 / 2 / 8 / 48 30 / 21 / 14 / 18.)
int splits(const PagedKv& kv, const PagedBatch& b, int heads) {
    if (few(kv, b, heads)) return 1;
    const int64_t max_len = b.max_pages * kv.page, keys = many_keys(kv.head_dim), blocks = (max_len + keys - 1) / keys;
    const int64_t n = (b.t + b.nseq - 1) / b.nseq, tiles = (n * (heads / kv.kv_heads) + 31) / 32;
    // Blocks before the new tokens are seen by all of them, others by half.
    const double seen = (blocks + double(std::max<int64_t>(max_len - n, 0)) / keys) / 2 * tiles, share = b.nseq > 1 ? 0.75 : 1.0;
    const double per_place = share * b.nseq * kv.kv_heads / (kv.head_dim == 64 ? 1024 : kv.head_dim == 128 ? 768 : 512);
    const double tile_us = 0.4 + kv.head_dim * 0.0057;
    int best = 1;
    double best_us = 1e30;
    for (const int k : {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32, 48}) {
        if (tiles < k) break;
        const double longest = double((tiles + k - 1) / k) + 4, all = (seen + 4.0 * k * blocks) * per_place;
        const double us = std::max(longest, all + longest / 4) * tile_us + (k > 1 ? 5 + 0.1 * k : 0);
        if (us < best_us) best_us = us, best = k;
    }
    return best;
}

int64_t part_bytes(const PagedKv& kv, const PagedBatch& b, int heads) {
    const int64_t n = splits(kv, b, heads);
    return n == 1 ? 0 : n * b.nseq * kv.kv_heads * b.max_pages * kv.page * 4;
}

template <typename T, int D>
void launch_d(hipStream_t s, Args a) {
    const int64_t lists = a.b.nseq * a.kv.kv_heads;
    if (few(a.kv, a.b, a.x.heads)) {
        // Chunks of 64 keys (of 64-wide heads 128) and more: 64 workgroups a CU are
        // enough.  (512 lists of 8,192 rows in 32 / 16 / 8 chunks 170 / 174 / 185 us.
        // The table's rows are counted, not the sequences': the same lists in a table
        // four times as wide, in chunks of 1,024, 476.)
        a.chunk = 4 * (D >= 128 ? 16 : 32);
        while (a.chunk < 4096 && lists * (a.max_len / a.chunk) > 16384) a.chunk *= 2;
        a.blocks = (a.max_len + a.chunk - 1) / a.chunk;
        if (lists * a.blocks >= MAX_BLOCKS) fail(E_CAPACITY, "attention_weights: too many work items");
        weights_few_kernel<T, D><<<dim3(unsigned(lists * a.blocks)), dim3(256), 0, s>>>(a);
        OMG_HIP(hipGetLastError());
        return;
    }
    a.blocks = (a.max_len + Many<T, D>::KEYS - 1) / Many<T, D>::KEYS;
    const int64_t n = lists * a.blocks * a.splits;
    if (n >= MAX_BLOCKS || (a.splits > 1 && lists > 65535)) fail(E_CAPACITY, "attention_weights: too many work items");
    constexpr unsigned lds = Many<T, D>::BUFS * (Many<T, D>::TILE * 2 + 4 * WAVE * 4);
    static std::atomic<uint64_t> lds_set{0};  // the devices, once per instantiation
    int device = 0;
    OMG_HIP(hipGetDevice(&device));
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device > 63 || !(lds_set.load(std::memory_order_relaxed) & bit)) {
        OMG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(weights_many_kernel<T, D>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
        lds_set.fetch_or(bit, std::memory_order_relaxed);
    }
    weights_many_kernel<T, D><<<dim3(unsigned(n)), dim3(256), lds, s>>>(a);
    OMG_HIP(hipGetLastError());
    if (a.splits > 1) {
        weights_join_kernel<<<dim3(unsigned((a.max_len + 255) / 256), unsigned(lists)), dim3(256), 0, s>>>(a);
        OMG_HIP(hipGetLastError());
    }
}

template <typename T>
void launch_t(hipStream_t s, const Args& a) {
    switch (a.kv.head_dim) {
        case 64: return launch_d<T, 64>(s, a);
        case 128: return launch_d<T, 128>(s, a);
        case 256: return launch_d<T, 256>(s, a);
        default: return launch_d<T, 512>(s, a);
    }
}

}  // namespace

int64_t attention_weights_workspace(const PagedKv& kv, const PagedBatch& b, int heads) {
    check(kv, b, heads);
    return part_bytes(kv, b, heads);
}

void launch_attention_weights(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const AttnWeights& x,
                              void* workspace, size_t bytes) {
    check(kv, b, x.heads);
    if (!x.q || !aligned16(x.q)) fail(E_INVALID, "attention_weights: q must be a 16-byte aligned device pointer");
    if (x.ldq < int64_t(x.heads) * kv.head_dim || x.ldq % 8)
        fail(E_INVALID, "attention_weights: ldq must hold the heads and be a multiple of 8");
    if (x.ldq > (1 << 24)) fail(E_INVALID, "attention_weights: ldq must be at most 2^24");
    if (!x.lse || !x.weights) fail(E_INVALID, "attention_weights: null lse or weights");
    if (x.ldw < b.max_pages * kv.page) fail(E_INVALID, "attention_weights: ldw must hold a sequence's rows");
    if (!(x.scale > 0.0f) || x.scale > 1e30f)
        fail(E_INVALID, "attention_weights: scale must be positive and finite");
    if (x.window < 0) fail(E_INVALID, "attention_weights: window must not be negative");
    const int64_t need = part_bytes(kv, b, x.heads);
    if (int64_t(bytes) < need)
        fail(E_CAPACITY, "attention_weights: the workspace needs " + std::to_string(need) + " bytes");
    if (need && (!workspace || !aligned16(workspace)))
        fail(E_INVALID, "attention_weights: the workspace must be 16-byte aligned");
    Args a{};
    a.kv = kv, a.b = b, a.x = x;
    a.hpg = x.heads / kv.kv_heads;
    a.page_shift = log2_of(kv.page);
    a.max_len = b.max_pages * kv.page;
    a.splits = splits(kv, b, x.heads);
    a.part = need ? static_cast<float*>(workspace) : nullptr;
    kv.dtype == ELEM_F16 ? launch_t<half_t>(s, a) : launch_t<bf16_t>(s, a);
}

}  // namespace omg
