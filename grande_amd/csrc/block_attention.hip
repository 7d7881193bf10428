// Attention over few blocks: a token's own page and, of the pages before it,
// those whose mean keys score highest against its queries.
//
//   mean[p]    = mean of the rows of page p                    (block_means)
//   score[b]   = sum over a KV head's query heads of q . mean  (block_scores)
//   chosen     = the token's own block and the best others     (block_choose)
//   out        = softmax over the chosen blocks' rows          (attention_blocks)
//
// Means and scores are sums in 64 bits, rounded to f32 once: which block is
// taken hangs on them, and so it does not hang on the order of a sum (one in
// some 10^9 rounds the other way).  A score is linear in the queries, so that a
// KV head's query heads come in as their sum; the products run on
// v_mfma_f64_16x16x4.
//
// The last step is shared_attention.h's own-key items with a list of pages in
// the place of a sequence's table.
#include "choose.h"
#include "shared_attention.h"

namespace omg {

namespace {

typedef double doublex4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------- means

struct MeanArgs {
    PagedKv kv;
    PagedBatch b;
    float* means;
    int page_shift;
    int64_t max_len;
};

// A workgroup a page and KV head: the pages of the batch's new rows, found by
// bounds start[s] / page + 2 s that leave each sequence enough of them.  A lane
// sums 8 head dims of every (4 * 512 / D)-th row.  A step's new rows lie in a page
// or two a sequence: a launch and two dependent loads, 4.4 to 5 us for 12 to 64
// sequences.
template <typename T, int D>
__global__ __launch_bounds__(256) void block_means_kernel(MeanArgs a) {
    constexpr int L = D / 8, W = WAVE / L, ROWS = 4 * W;  // rows at once
    __shared__ double sums[ROWS][D + 2];
    const int tid = int(threadIdx.x), lane = tid % WAVE;
    const int g = int(blockIdx.x % a.kv.kv_heads);
    const int64_t item = blockIdx.x / a.kv.kv_heads;
    int64_t s = item, index = 0, n = 1;
    if (a.b.start) {
        int64_t lo = 0, left = a.b.nseq;
        while (left > 0) {
            const int64_t step = (left + WAVE - 1) / WAVE, k = lo + (lane + 1) * step, at = k <= lo + left ? k : lo + left;
            const int cnt = __popcll(__ballot(k <= lo + left && (int64_t(a.b.start[at]) >> a.page_shift) + 2 * at <= item));
            const int64_t rest = left - cnt * step;
            lo += cnt * step;
            left = rest < step - 1 ? rest : step - 1;
        }
        s = lo;
        if (s >= a.b.nseq) return;
        index = item - (int64_t(a.b.start[s]) >> a.page_shift) - 2 * s;
        n = a.b.start[s + 1] - a.b.start[s];
    }
    const int64_t len = a.b.lens[s] < a.max_len ? a.b.lens[s] : a.max_len;
    const int64_t from = a.b.lens[s] - n < 0 ? 0 : a.b.lens[s] - n;  // the first new row
    const int64_t i = (from >> a.page_shift) + index;
    if (index < 0 || n <= 0 || i << a.page_shift >= len) return;
    const int64_t p = a.b.table[s * a.b.table_ld + i];
    if (p < 0 || p >= a.kv.npages) return;
    const int64_t rest = len - (i << a.page_shift);
    const int rows = int(rest < a.kv.page ? rest : a.kv.page), c = lane % L * 8, r0 = tid / L;
    const T* k = static_cast<const T*>(a.kv.k) + p * a.kv.page_stride + int64_t(g) * a.kv.page * D + c;
    double sum[8] = {};
#pragma unroll 4
    for (int r = r0; r < rows; r += ROWS) {
        float x[8];
        load8(k + int64_t(r) * D, x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += double(x[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[r0][c + e] = sum[e];
    __syncthreads();
    for (int d = tid; d < D; d += 256) {
        double v = 0.0;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) v += sums[r][d];
        a.means[(p * a.kv.kv_heads + g) * D + d] = float(v / rows);
    }
}

// ------------------------------------------------------------------ scores

struct BlockArgs {
    Args a;
    const float* means;
    float* scores;     // [t][kv_heads][blocks_ld]
    int64_t blocks_ld;
    int32_t* chosen;   // [t][kv_heads][keep]
    int keep;          // blocks of a token
    int np;            // blocks of the prefix
    int chunk;         // entries of a work item
    int64_t prefix_items, own_chunks;
};

// 16 tokens (of any sequences: prefix blocks; of one: its own) x 64 blocks, 16
// a wave; FEW: x 16, a quarter of the head dims a wave.  The queries' sums lie in
// LDS in the order in which the lanes take them: lane l of a step holds token l %
// 16 and dims of the quarter l / 16 of the head, and blocks' means likewise, a run
// of 16 bytes at a time.  Bound by the f64 products and the loads' latency before
// them: 64 tokens x 8 KV heads of 128 on some 1,050 blocks 12 us, 12 x 4 of 256 on
// 126 5.9.
template <typename T, int D, bool FEW>
__global__ __launch_bounds__(256) void block_scores_kernel(BlockArgs x) {
    constexpr int Q = D / 4, QW = FEW ? Q / 4 : Q;  // dims of a quarter, of them a wave's
    constexpr int DC = FEW || Q < 64 ? Q : 64;      // of a quarter in LDS at once
    constexpr int BW = FEW ? 16 : 64;               // blocks
    __shared__ double qs[DC * WAVE > 1024 ? DC * WAVE : 1024];
    const Args& a = x.a;
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int G = a.kv.kv_heads;
    int64_t id = blockIdx.x;
    const int g = int(id % G);
    id /= G;
    // The item's tokens t0 .. t1 - 1, blocks b0 .. of a table and their place in the scores.
    int64_t t0, t1, b0, nblocks, first;
    const int32_t* table;
    if (id < x.prefix_items) {
        const int64_t chunks = (x.np + BW - 1) / BW;
        t0 = id / chunks * 16, t1 = t0 + 16 < a.b.t ? t0 + 16 : a.b.t;
        b0 = id % chunks * BW, nblocks = x.np, first = 0, table = a.b.prefix_table;
    } else {
        id -= x.prefix_items;
        const int64_t i = id / x.own_chunks;
        int64_t s = i, tile = 0, end;
        t0 = i, end = i + 1;
        if (a.b.start) {
            // tile i is of the sequence with start[s] / 16 + s <= i
            int64_t lo = 0, left = a.b.nseq;
            while (left > 0) {
                const int64_t step = (left + WAVE - 1) / WAVE, k = lo + (lane + 1) * step, at = k <= lo + left ? k : lo + left;
                const int cnt = __popcll(__ballot(k <= lo + left && int64_t(a.b.start[at]) / 16 + at <= i));
                const int64_t rest = left - cnt * step;
                lo += cnt * step;
                left = rest < step - 1 ? rest : step - 1;
            }
            s = lo;
            if (s >= a.b.nseq) return;
            tile = i - int64_t(a.b.start[s]) / 16 - s;
            t0 = a.b.start[s] + 16 * tile, end = a.b.start[s + 1];
        }
        t1 = t0 + 16 < end ? t0 + 16 : end;
        if (t1 > a.b.t) t1 = a.b.t;  // (token rows outside the batch's are nobody's)
        if (tile < 0 || t0 >= t1 || t1 <= 0) return;
        // (blocks up to the last token's own have a score that counts)
        const int64_t row = int64_t(a.b.lens[s]) - (end - (t1 - 1));
        const int64_t have = row < 0 ? 0 : (row >> a.page_shift) + 1;
        b0 = id % x.own_chunks * BW, nblocks = have < a.b.max_pages ? have : a.b.max_pages, first = x.np;
        table = a.b.table + s * a.b.table_ld;
    }
    if (b0 >= nblocks) return;
    b0 += FEW ? 0 : wave * 16;             // the wave's
    const int64_t mine = b0 + lane % 16;  // the block whose means the lane loads
    const int64_t p = mine < nblocks ? table[mine] : -1;
    const bool there = p >= 0 && p < a.kv.npages;
    // (a page that is not there: the first page's means, and no score from them)
    const float* mean = x.means + ((there ? p : 0) * G + g) * D + lane / 16 * Q + (FEW ? wave * QW : 0);
    constexpr int N = QW < 32 ? QW : 32;  // dims whose means are under way
    float4 m[N / 4];
#pragma unroll
    for (int d = 0; d < N; d += 4) m[d / 4] = *reinterpret_cast<const float4*>(mean + d);
    doublex4 acc = {0.0, 0.0, 0.0, 0.0};
    for (int c = 0; c < Q; c += DC) {
        if (c) __syncthreads();
        // A thread sums 8 dims of a token over the heads, IT times.
        constexpr int IT = DC < 32 ? 1 : DC / 32, HB = IT < 4 ? 4 : 2;
        const int tok = tid % 16, quarter = tid / 16 % 4;
        double sum[IT][8] = {};
        if (t0 + tok >= 0 && t0 + tok < t1 && wave * 8 < DC) {
            const T* q = static_cast<const T*>(a.x.q) + (t0 + tok) * a.x.ldq + int64_t(g) * a.hpg * D + quarter * Q + c + wave * 8;
            for (int h0 = 0; h0 < a.hpg; h0 += HB) {
                float v[IT][HB][8];
#pragma unroll
                for (int i = 0; i < IT; ++i)
#pragma unroll
                    for (int h = 0; h < HB; ++h) load8(q + int64_t(h0 + h < a.hpg ? h0 + h : h0) * D + 32 * i, v[i][h]);
#pragma unroll
                for (int i = 0; i < IT; ++i)
#pragma unroll
                    for (int h = 0; h < HB; ++h)
#pragma unroll
                        for (int e = 0; e < 8; ++e) sum[i][e] += h0 + h < a.hpg ? double(v[i][h][e]) : 0.0;
            }
        }
        if (wave * 8 < DC) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) qs[(wave * 8 + 32 * i + e) * WAVE + quarter * 16 + tok] = sum[i][e];
        }
        __syncthreads();
#pragma unroll
        for (int d0 = 0; d0 < (FEW ? QW : DC); d0 += N) {
            float4 next[N / 4];
            const bool more = c + d0 + N < QW;
            if (more) {
#pragma unroll
                for (int d = 0; d < N; d += 4) next[d / 4] = *reinterpret_cast<const float4*>(mean + c + d0 + N + d);
            }
#pragma unroll
            for (int d = 0; d < N; d += 4) {
                const double* q = qs + ((FEW ? wave * QW : 0) + d0 + d) * WAVE + lane;
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(double(m[d / 4].x), q[0], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(double(m[d / 4].y), q[WAVE], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(double(m[d / 4].z), q[2 * WAVE], acc, 0, 0, 0);
                acc = __builtin_amdgcn_mfma_f64_16x16x4f64(double(m[d / 4].w), q[3 * WAVE], acc, 0, 0, 0);
            }
            if (more) {
#pragma unroll
                for (int d = 0; d < N / 4; ++d) m[d] = next[d];
            }
        }
    }
    // The lane has blocks 4 r + lane / 16 of the wave's, token lane % 16; FEW: the
    // sum of all waves' for r = wave.
    if constexpr (FEW) {
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) qs[(wave * 4 + r) * WAVE + lane] = acc[r];
        __syncthreads();
        double v = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v += qs[(i * 4 + wave) * WAVE + lane];
        acc[0] = v;
    }
    const uint64_t gone = __ballot(!there) & 0xffff;
    const int64_t tok = t0 + lane % 16;
    if (tok < 0 || tok >= t1) return;
#pragma unroll
    for (int i = 0; i < (FEW ? 1 : 4); ++i) {
        const int of = 4 * (FEW ? wave : i) + lane / 16;
        if (b0 + of < nblocks)
            x.scores[(tok * G + g) * x.blocks_ld + first + b0 + of] = gone >> of & 1 ? 0.0f : float(acc[i]);
    }
}

// ------------------------------------------------------------------ choose

// The block of a token's own row (below zero: it sees nothing), counted from
// the prefix's first.  A length past the table: the table's last row.
__device__ inline int own_block(const BlockArgs& x, const SeqRow& at) {
    if (at.seq < 0 || at.row < 0) return -1;
    const int64_t row = at.row < x.a.max_len ? at.row : x.a.max_len - 1;
    return x.np + int(row >> x.a.page_shift);
}

constexpr int CHOOSE_T = 256;

// put(rank, block) for the blocks that a token takes, all threads of the
// workgroup together; largest(n, k, hand) hands out the k best of the first n.
template <typename L, typename F>
__device__ inline void choose_blocks(const BlockArgs& x, int own, L largest, F put) {
    const int tid = int(threadIdx.x), others = own < x.keep - 1 ? own : x.keep - 1;
    if (others == own) {
        for (int i = tid; i < own; i += CHOOSE_T) put(i, i);
    } else {
        largest(own, uint32_t(others), [&](int rank, int b, float) { put(rank, b); });
    }
    for (int i = others + tid; i < x.keep; i += CHOOSE_T) put(i, i == others ? own : -1);
}

// A workgroup a token and KV head, of 256 threads, so that many lists share a CU
// (a step's 512 lists of 1,000 blocks: 9 us; 48 of 126: 5 to 6 us, the choice's
// chain of barriers).
template <bool HELD>
__global__ __launch_bounds__(CHOOSE_T) void block_choose_kernel(BlockArgs x) {
    typedef Choose<CHOOSE_T, HELD> C;
    __shared__ typename C::Shared shared;
    const int tid = int(threadIdx.x);
    const int64_t list = blockIdx.x, tok = list / x.a.kv.kv_heads;
    const SeqRow at = token_row(x.a.b, tok, tid % WAVE);
    const int own = own_block(x, at);
    int32_t* to = x.chosen + list * x.keep;
    if (own < 0) {
        if (at.seq >= 0)  // (rows that no sequence has stay as they are)
            for (int i = tid; i < x.keep; i += CHOOSE_T) to[i] = -1;
        return;
    }
    auto largest = [&](int n, uint32_t k, auto hand) { C::run(shared, x.scores + list * x.blocks_ld, n, k, hand); };
    choose_blocks(x, own, largest, [&](int rank, int b) { to[rank] = b; });
}

// --------------------------------------------------------------- attention

// 16 query rows of a token and KV head over up to 64 entries of its list: each
// wave every fourth 16-key tile.  All rows see the same keys.  (512 lists of 64 x
// 64 rows, 128-wide: 82 us, 1.1 GB through L2 and 270 MB from HBM; a second tile
// a wave under way 85.)
// CHOOSE: the workgroup makes its list's choice itself, each split and part of the
// heads again.
template <typename T, int D, bool CHOOSE>
__global__ __launch_bounds__(NW * 64, D == 512 ? 1 : D == 64 ? 4 : 2) void attention_blocks_kernel(BlockArgs x) {
    typedef Core<T, D, WAVES_KEYS> C;
    extern __shared__ __attribute__((aligned(1024))) unsigned char smem_raw[];
    const Args& a = x.a;
    T* smem = reinterpret_cast<T*>(smem_raw);
    const int tid = int(threadIdx.x), lane = tid % WAVE, wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int G = a.kv.kv_heads, parts = (a.hpg + 15) / 16;
    int64_t id = blockIdx.x;
    const int g = int(id % G);
    id /= G;
    const int split = uni(int(id % a.p.os));
    id /= a.p.os;
    const int64_t tok = id / parts;
    const int head0 = int(id - tok * parts) * 16 + lane % 16;
    const int64_t list = tok * G + g;
    float score = 0.0f;  // CHOOSE: of few blocks the thread's, on its way before their number is known
    if (CHOOSE && x.blocks_ld <= CHOOSE_T && tid < x.blocks_ld) score = x.scores[list * x.blocks_ld + tid];
    const SeqRow at = token_row(a.b, tok, lane);
    if (at.seq < 0) return;
    const int own = own_block(x, at);
    Row r{head0 < a.hpg, int(tok * a.x.heads + g * a.hpg + head0), int(at.seq), 0};
    C core;
    core.init(r.valid ? static_cast<const T*>(a.x.q) + tok * a.x.ldq + int64_t(g * a.hpg + head0) * D : nullptr, lane);

    // Lane e: the page of the item's entry e and its rows that the token sees.
    const int e0 = split * x.chunk, count = imin(x.chunk, x.keep - e0);
    int block = -1;
    if constexpr (CHOOSE) {
        typedef Choose<CHOOSE_T, true> Best;
        static_assert(CHOOSE_T == NW * 64 && sizeof(typename Best::Shared) <= NW * 16 * D * 4, "the tiles' place");
        auto& shared = *reinterpret_cast<typename Best::Shared*>(smem_raw);
        __shared__ int taken[WAVE];
        int32_t* to = x.chosen && split == 0 && id % parts == 0 ? x.chosen + list * x.keep : nullptr;
        auto put = [&](int rank, int b) {
            if (rank >= e0 && rank < e0 + count) taken[rank - e0] = b;
            if (to) to[rank] = b;
        };
        if (own >= 0)
            choose_blocks(x, own, [&](int n, uint32_t k, auto hand) {
                if (x.blocks_ld <= CHOOSE_T)
                    Best::run_few(shared, score, n, k, hand);
                else
                    Best::run(shared, x.scores + list * x.blocks_ld, n, k, hand);
            }, put);
        else
            for (int i = tid; i < x.keep; i += CHOOSE_T) put(i, -1);
        __syncthreads();
        if (lane < count) block = taken[lane];
    } else if (lane < count) {
        block = x.chosen[list * x.keep + e0 + lane];
    }
    int page = -1, rows = 0;
    if (block >= 0 && block <= own) {
        const int P = int(a.b.prefix_len), j = block - x.np;
        page = j < 0 ? a.b.prefix_table[block] : a.b.table[at.seq * a.b.table_ld + j];
        rows = j < 0 ? imin(a.kv.page, P - (block << a.page_shift))
                     : int(at.row - (int64_t(j) << a.page_shift) < a.kv.page ? at.row - (int64_t(j) << a.page_shift) + 1 : a.kv.page);
        if (unsigned(page) >= unsigned(a.kv.npages)) rows = 0;
    }
    const Stream<T, D, WAVES_KEYS> st{a, g, wave, lane, smem};
    const int per = a.kv.page / 16;  // tiles of a block
    const int tiles = uni(__popcll(__ballot(block >= 0))) * per;
    for (int k = wave; k < tiles; k += NW) {
        const int e = k / per, r0 = (k - e * per) * 16;
        const int pg = __builtin_amdgcn_readlane(page, e), lim = __builtin_amdgcn_readlane(rows, e);
        if (r0 >= lim) continue;
        st.issue(r0, lim, st.buf(0), pg, pg);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        core.tile(uint32_t(uintptr_t((lds_ptr)st.buf(0))), lane, r0, lim - r0 >= 16, 0, r.valid ? lim : 0, 0, a.c);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    emit_keys<T, D>(a, core, r, lane, wave, split, reinterpret_cast<float*>(smem_raw), [&](uint64_t bad, float lg) {
        seen_alone<T, D>(a, g, r, bad, lg, lane, split, wave, [&](int, auto keys) {
            for (int e = 0; e < count; ++e) {
                const int pg = __builtin_amdgcn_readlane(page, e), lim = __builtin_amdgcn_readlane(rows, e);
                keys(0, lim, [&](int) { return int64_t(pg); });
            }
        });
    });
}

// -------------------------------------------------------------------- host

struct BlockPlan {
    int64_t np, blocks;  // blocks of the prefix, and of a sequence with it
    int chunk, splits;
    int64_t scores, chosen, parts;  // bytes of the workspace's regions
};

void check_blocks(const PagedKv& kv, const PagedBatch& b, int heads, int64_t keep) {
    check(kv, b, heads, "attention_blocks");
    if (keep <= 0 || keep > 4096) fail(E_INVALID, "attention_blocks: blocks must be 1 to 4096");
}

// Workgroups of attention_blocks_kernel that the chip takes at once, by LDS.
int64_t places(int head_dim) { return 256 * (head_dim == 64 ? 4 : head_dim == 512 ? 1 : 2); }

// Entries are split over work items until these fill the chip's places,
// at least 128 rows at a time and at most an entry a lane.  (26 blocks of 128 rows of
// 512: 13 items' launches 36 us in all, 26 32; 64 of 64 x 128 28 and 24.  Lists of one token
// each that start together stay together, and what one reads the next finds in
// L2: 512 lists as 1,024 items 116 us, as 512 82.)
BlockPlan plan_blocks(const PagedKv& kv, const PagedBatch& b, int heads, int64_t keep) {
    BlockPlan p{};
    p.np = (b.prefix_len + kv.page - 1) / kv.page;
    p.blocks = p.np + b.max_pages;
    const int64_t hpg = heads / kv.kv_heads, items = b.t * kv.kv_heads * ((hpg + 15) / 16);
    const int64_t least = (keep + 63) / 64, most = std::min<int64_t>(64, std::max<int64_t>(1, keep * kv.page / 128));
    const int64_t want = std::max(least, std::min(most, places(kv.head_dim) / items));
    p.chunk = int((keep + want - 1) / want);
    p.splits = int((keep + p.chunk - 1) / p.chunk);
    p.scores = up(b.t * kv.kv_heads * p.blocks * 4, 16);
    p.chosen = up(b.t * kv.kv_heads * keep * 4, 16);
    p.parts = p.splits > 1 ? p.splits * b.t * heads * (kv.head_dim * 4 + 4) : 0;
    return p;
}

template <typename T, int D, bool CHOOSE>
void launch_chosen(hipStream_t s, const BlockArgs& x, int64_t items) {
    constexpr unsigned lds = NW * 16 * D * 4 + 2 * NW * 16 * 4;  // tiles of K and V a wave; their join
    static std::atomic<uint64_t> lds_set{0};                     // the devices, once per instantiation
    int device = 0;
    OMG_HIP(hipGetDevice(&device));
    const uint64_t bit = uint64_t(1) << (device & 63);
    if (device > 63 || !(lds_set.load(std::memory_order_relaxed) & bit)) {
        OMG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(attention_blocks_kernel<T, D, CHOOSE>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
        lds_set.fetch_or(bit, std::memory_order_relaxed);
    }
    attention_blocks_kernel<T, D, CHOOSE><<<dim3(unsigned(items)), dim3(NW * 64), lds, s>>>(x);
    OMG_HIP(hipGetLastError());
}

template <typename T, int D>
void launch_blocks_d(hipStream_t s, BlockArgs x, int32_t* room) {
    const Args& a = x.a;
    const int64_t lists = a.b.t * a.kv.kv_heads;
    const int64_t items = lists * a.p.os * ((a.hpg + 15) / 16);
    const int64_t own_tiles = a.b.start ? a.b.t / 16 + a.b.nseq : a.b.nseq;
    auto scored = [&](int blocks) {  // items of so many blocks each
        x.prefix_items = (a.b.t + 15) / 16 * ((x.np + blocks - 1) / blocks);
        x.own_chunks = (a.b.max_pages + blocks - 1) / blocks;
        return (x.prefix_items + own_tiles * x.own_chunks) * a.kv.kv_heads;
    };
    // (56 items for 12 x 4 lists of 126 blocks, 256-wide, 8.1 us, of 16 blocks 5.8; 304
    // 10.6 and 7.0, 768 14.0 and 14.1; 1,024 of 128-wide heads 11.8 and 15.)
    const bool few = scored(64) < 768;
    const int64_t scores = scored(few ? 16 : 64);
    if (scores >= MAX_BLOCKS || items >= MAX_BLOCKS || lists >= MAX_BLOCKS)
        fail(E_CAPACITY, "attention_blocks: too many work items");
    few ? block_scores_kernel<T, D, true><<<dim3(unsigned(scores)), dim3(256), 0, s>>>(x)
        : block_scores_kernel<T, D, false><<<dim3(unsigned(scores)), dim3(256), 0, s>>>(x);
    OMG_HIP(hipGetLastError());
    // Work items that the chip takes at once choose for themselves (12 x 4 lists of
    // 126 blocks: 18 us for 15.5 and 6, 512 of 1,050: 87 for 82 and 9).  More of them
    // would hold the tiles' LDS through a chain of barriers, round by round (2,048 of
    // 196: 114 us, in two launches 97 and 12).
    const bool held = x.blocks_ld <= CHOOSE_R * CHOOSE_T;
    if (held && items <= places(D)) {
        launch_chosen<T, D, true>(s, x, items);
    } else {
        if (!x.chosen) x.chosen = room;
        held ? block_choose_kernel<true><<<dim3(unsigned(lists)), dim3(CHOOSE_T), 0, s>>>(x)
             : block_choose_kernel<false><<<dim3(unsigned(lists)), dim3(CHOOSE_T), 0, s>>>(x);
        OMG_HIP(hipGetLastError());
        launch_chosen<T, D, false>(s, x, items);
    }
    if (!a.part_o) return;
    const int64_t rows = a.b.t * a.x.heads;
    if (a.p.slots() > 8)
        attention_join_kernel<T, D, 4><<<dim3(unsigned(rows)), dim3(256), 0, s>>>(a);
    else
        attention_join_kernel<T, D, 1><<<dim3(unsigned((rows + 3) / 4)), dim3(256), 0, s>>>(a);
    OMG_HIP(hipGetLastError());
}

template <typename T>
void launch_blocks_t(hipStream_t s, const BlockArgs& x, int32_t* room) {
    switch (x.a.kv.head_dim) {
        case 64: return launch_blocks_d<T, 64>(s, x, room);
        case 128: return launch_blocks_d<T, 128>(s, x, room);
        case 256: return launch_blocks_d<T, 256>(s, x, room);
        default: return launch_blocks_d<T, 512>(s, x, room);
    }
}

template <typename T>
void launch_means_t(hipStream_t s, const MeanArgs& a, unsigned blocks) {
    switch (a.kv.head_dim) {
        case 64: block_means_kernel<T, 64><<<dim3(blocks), dim3(256), 0, s>>>(a); break;
        case 128: block_means_kernel<T, 128><<<dim3(blocks), dim3(256), 0, s>>>(a); break;
        case 256: block_means_kernel<T, 256><<<dim3(blocks), dim3(256), 0, s>>>(a); break;
        default: block_means_kernel<T, 512><<<dim3(blocks), dim3(256), 0, s>>>(a);
    }
    OMG_HIP(hipGetLastError());
}

}  // namespace

void launch_block_means(hipStream_t s, const PagedKv& kv, const PagedBatch& b, float* means) {
    check_kv(kv, "block_means");
    check_batch(b, kv, "block_means");
    if (!means || !aligned16(means)) fail(E_INVALID, "block_means: means must be a 16-byte aligned device pointer");
    const int64_t items = (b.start ? b.t / kv.page + 2 * b.nseq : b.nseq) * kv.kv_heads;
    if (items >= MAX_BLOCKS) fail(E_CAPACITY, "block_means: too many rows for one call");
    const MeanArgs a{kv, b, means, log2_of(kv.page), b.max_pages * kv.page};
    kv.dtype == ELEM_F16 ? launch_means_t<half_t>(s, a, unsigned(items)) : launch_means_t<bf16_t>(s, a, unsigned(items));
}

int64_t attention_blocks_workspace(const PagedKv& kv, const PagedBatch& b, int heads, int64_t keep) {
    check_blocks(kv, b, heads, keep);
    const BlockPlan p = plan_blocks(kv, b, heads, keep);
    return p.scores + p.chosen + p.parts;
}

void launch_attention_blocks(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const SharedAttn& x,
                             const float* means, int64_t keep, int32_t* chosen, void* workspace, size_t bytes) {
    check_blocks(kv, b, x.heads, keep);
    check_rows(kv, x, "attention_blocks");
    if (!means || !aligned16(means)) fail(E_INVALID, "attention_blocks: means must be a 16-byte aligned device pointer");
    const BlockPlan p = plan_blocks(kv, b, x.heads, keep);
    const int64_t need = p.scores + p.chosen + p.parts;
    if (int64_t(bytes) < need)
        fail(E_CAPACITY, "attention_blocks: the workspace needs " + std::to_string(need) + " bytes");
    if (!workspace || !aligned16(workspace)) fail(E_INVALID, "attention_blocks: the workspace must be 16-byte aligned");
    char* room = static_cast<char*>(workspace);
    BlockArgs k{};
    k.a.kv = kv, k.a.b = b, k.a.x = x;
    k.a.p.os = p.splits;  // (slots for the join)
    k.a.hpg = x.heads / kv.kv_heads;
    k.a.page_shift = log2_of(kv.page);
    k.a.max_len = b.max_pages * kv.page;
    k.a.c = x.scale * 1.4426950408889634f;
    if (p.parts) {
        k.a.part_o = reinterpret_cast<float*>(room + p.scores + p.chosen);
        k.a.part_lg = k.a.part_o + p.splits * b.t * x.heads * kv.head_dim;
    }
    k.means = means;
    k.scores = reinterpret_cast<float*>(room), k.blocks_ld = p.blocks;
    k.chosen = chosen;
    k.keep = int(keep), k.np = int(p.np), k.chunk = p.chunk;
    int32_t* list = reinterpret_cast<int32_t*>(room + p.scores);
    kv.dtype == ELEM_F16 ? launch_blocks_t<half_t>(s, k, list) : launch_blocks_t<bf16_t>(s, k, list);
}

}  // namespace omg
