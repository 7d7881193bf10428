// Attention of drafted tokens, which see the rows before them and, of the
// sequence's new rows, those that their masks name: the kernels of
// shared_attention.h with MASKED.  Only tiles that hold new rows look at the
// masks (a word or two a lane, asked for a tile ahead).  Measured, and what bounds it:
//   12 drafts of 4 to 8 tokens x 4 heads of 256 on 2,000 shared keys (f16): 12.5 us
//     and the join's 4: latency.
//   208 of 7 to 13 tokens x 8 heads of 256 on 8,000: 192 to 201 us a call in a row,
//     about 700 TFLOP/s (traced one by one 202 and, the slots' join, 17): a wave's
//     chain of product, softmax and product, two waves a SIMD; MFMAs 39 % and vector
//     instructions 35 % of the busy SIMDs' cycles, and 396 items on 512 places.
//   16 trees of 31 to 61 tokens x 32 heads of 128 on 32,749 (bf16): 517 to 542 us a
//     call in a row, cards differ, 800 TFLOP/s (traced one by one 563 to 612 and 17):
//     vector instructions 50 %, MFMAs 42 % of the busy SIMDs' cycles.
#include "shared_attention.h"

namespace omg {

namespace {

// The tile and the splits of least time by a model of the launch: a work item
// takes so long a tile of keys (a chain of dependent steps: hardly longer with
// two or three workgroups on the CU) and two tiles' time besides; the places
// that the chip has take items one after the other, the last ones of them for half
// a round (a whole round: 90 trees of 26 tokens x 32 heads of 128 on 1,323 + 590 keys in
// three splits' rounds 172 us, in one item each 130); a slot of partial results is
// written and read.  Measured, for 32 and 16 rows a wave: 1.76 and 0.97 us a tile of
// 256-wide heads, 1.24 and 0.67 of 128-wide ones.  (One split of the 8,000 keys
// for 2,100 tokens x 8 heads of 256, 132 items, 459 us, three 189; the best at 16
// rows a wave 280.  70 tokens x 4 heads on 2,000 keys 17 us at 32 rows, 13 at
// 16.)
//
// With a window the prefix counts as far as it reaches, in at most `most` slots (a
// workspace's size does not hang on the window): 20 trees of 21 tokens x 15 heads of
// 64 on 14,304 keys at 1,024 40 -> 24 us, where the splits were the prefix's.
Plan plan_tree(const PagedKv& kv, const PagedBatch& b, int heads, int window = 0, int64_t most = INT64_MAX) {
    const Plan from = plan(kv, b, heads);
    const int64_t hpg = heads / kv.kv_heads, rows = b.t * hpg, max_len = b.max_pages * kv.page;
    const int64_t P = window > 0 ? std::min<int64_t>(b.prefix_len, window) : b.prefix_len;
    const int D = kv.head_dim;
    const double slot_us = double(b.t) * heads * D * 8 / 4.5e6;
    auto chunk = [](int64_t keys, int64_t n) { return up((keys + n - 1) / n, 32); };
    static constexpr int splits[] = {1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 32, 48, 64};
    Plan best = from;
    double best_us = 1e30;
    for (const int tile : {int(WAVES_16), int(WAVES_32)}) {
        if (from.tile == WAVES_KEYS || (tile == WAVES_32 && D == 512)) continue;
        Plan q = from;
        q.tile = tile;
        const int64_t M = tile == WAVES_16 ? 64 : 128;
        q.ntile = int((rows + M - 1) / M);
        const int64_t base = q.ntile * int64_t(kv.kv_heads);
        const int KT = D == 512 ? 16 : 32;
        const double tile_us = (0.7 + D / 240.0) * (tile == WAVES_16 ? 0.55 : 1.0);
        const int64_t places = 256 * (D == 64 ? 4 : D == 128 ? 3 : D == 512 && !q.fused ? 1 : 2);
        auto tiles = [&](int64_t keys) { return double((keys + KT - 1) / KT) + 2; };
        auto take = [&](const Plan& p, double longest) {
            const int64_t nsplit = p.whole ? 1 : p.np + (p.fused ? p.os : 0);
            if (p.slots() > most) return;
            const double full = double(base * nsplit) / places, rounds = full > 1.0 ? full + 0.5 : 1.0;
            const double us = rounds * longest * tile_us + (p.slots() > 1 ? 3.0 + slot_us * p.slots() : 0.0);
            if (us < best_us) best_us = us, best = p;
        };
        if (!q.fused) {  // (the own keys' items as they are)
            if (P == 0) take(q, 0);
            for (const int n : splits) {
                if (P == 0) break;
                q.chunk_p = int(chunk(P, n)), q.np = int((P + q.chunk_p - 1) / q.chunk_p);
                take(q, tiles(q.chunk_p));
            }
            continue;
        }
        // A tile runs through the own keys of each sequence that it holds.
        const int64_t held = std::min<int64_t>(b.nseq, M * b.nseq / rows + 2);
        q.whole = true, q.np = 0, q.chunk_p = 0, q.os = 1, q.chunk_o = int(std::min<int64_t>(up(max_len, 32), INT_MAX / 2));
        take(q, tiles(P) + held * tiles(max_len));
        q.whole = false;
        for (const int n : splits) {
            if (P == 0 && n > 1) break;
            if (P > 0) q.chunk_p = int(chunk(P, n)), q.np = int((P + q.chunk_p - 1) / q.chunk_p);
            for (int os = 1; os <= 64; os *= 4) {
                q.chunk_o = int(std::min<int64_t>(chunk(max_len, os), INT_MAX / 2));
                q.os = int((max_len + q.chunk_o - 1) / q.chunk_o);
                take(q, std::max(P > 0 ? tiles(q.chunk_p) : 0.0, held * tiles(std::min<int64_t>(q.chunk_o, max_len))));
            }
        }
    }
    return best;
}

}  // namespace

int64_t attention_tree_workspace(const PagedKv& kv, const PagedBatch& b, int heads) {
    check(kv, b, heads, "attention_tree");
    return part_bytes(plan_tree(kv, b, heads), kv, b, heads);
}

void launch_attention_tree(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const SharedAttn& x,
                           const TreeMask& tree, void* workspace, size_t bytes) {
    if (!tree.mask || reinterpret_cast<uintptr_t>(tree.mask) % 4)
        fail(E_INVALID, "attention_tree: mask must be a 4-byte aligned device pointer");
    if (tree.words <= 0 || tree.words > (1 << 20)) fail(E_INVALID, "attention_tree: mask_ld must be 1 to 2^20 words");
    if (x.window > 0 && !tree.positions) fail(E_INVALID, "attention_tree: a window needs the tokens' positions");
    if (reinterpret_cast<uintptr_t>(tree.positions) % 4) fail(E_INVALID, "attention_tree: positions must be 4-byte aligned");
    auto planned = [&](const PagedKv& kv, const PagedBatch& b, int heads) {
        const Plan p = plan_tree(kv, b, heads);
        return x.window > 0 && p.tile != WAVES_KEYS ? plan_tree(kv, b, heads, x.window, p.slots()) : p;
    };
    launch_attention<true>(s, kv, b, x, tree, planned, workspace, bytes, "attention_tree");
}

}  // namespace omg
