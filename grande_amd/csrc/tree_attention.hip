// Attention of drafted tokens, which see the rows before them and, of the
// sequence's new rows, those that their masks name: the kernels of
// shared_attention.h with MASKED.  Only tiles that hold new rows look at the
// masks (a word or two a lane, asked for a tile ahead).
#include "shared_attention.h"

namespace omg {

namespace {

// The splits of least time by a model of the launch: a work item takes so long
// a tile of keys (a chain of dependent steps: hardly longer with two or three
// workgroups on the CU) and two tiles' time besides; the places that the chip
// has take items in rounds; a slot of partial results is written and read.
Plan plan_tree(const PagedKv& kv, const PagedBatch& b, int heads) {
    Plan p = plan(kv, b, heads);  // the tile shape and whether own keys go into its tiles
    const int64_t hpg = heads / kv.kv_heads, rows = b.t * hpg, max_len = b.max_pages * kv.page, P = b.prefix_len;
    const int64_t M = p.tile == WAVES_KEYS ? 16 : p.tile == WAVES_16 ? 64 : 128;
    const int64_t base = p.ntile * int64_t(kv.kv_heads);
    const int D = kv.head_dim, KT = p.tile == WAVES_KEYS || D == 512 ? 16 : 32;
    const double tile_us = 0.7 + D / 240.0, slot_us = double(b.t) * heads * D * 8 / 4.5e6;
    const int64_t places = 256 * (D == 64 ? 4 : D == 128 ? 3 : D == 512 && !p.fused ? 1 : 2);
    auto tiles = [&](int64_t keys) { return double((keys + KT - 1) / KT) / (p.tile == WAVES_KEYS ? NW : 1) + 2; };
    auto chunk = [](int64_t keys, int64_t n) { return up((keys + n - 1) / n, 32); };
    double best = 1e30;
    const Plan from = p;
    if (p.fused) {
        // A tile runs through the own keys of the sequences it holds.
        const int64_t held = std::min<int64_t>(b.nseq, M * b.nseq / rows + 2);
        auto take = [&](Plan q, double items, double most) {
            const double t = std::max(1.0, std::ceil(items / places)) * most * tile_us +
                             (q.whole ? 0.0 : 3.0 + slot_us * (q.np + q.os));
            if (t < best) best = t, p = q;
        };
        Plan q = from;
        q.whole = true, q.np = 0, q.chunk_p = 0, q.os = 1, q.chunk_o = int(std::min<int64_t>(up(max_len, 32), INT_MAX / 2));
        take(q, double(base), tiles(P) + held * tiles(max_len));
        q.whole = false;
        for (int np = P > 0 ? 1 : 0; np <= (P > 0 ? 64 : 0); ++np) {
            if (np) q.chunk_p = int(chunk(P, np)), q.np = int((P + q.chunk_p - 1) / q.chunk_p);
            for (int os = 1; os <= 64; os *= 2) {
                q.chunk_o = int(std::min<int64_t>(chunk(max_len, os), INT_MAX / 2));
                q.os = int((max_len + q.chunk_o - 1) / q.chunk_o);
                take(q, double(base) * (q.np + q.os),
                     std::max(np ? tiles(q.chunk_p) : 0.0, held * tiles(std::min<int64_t>(q.chunk_o, max_len))));
            }
        }
        return p;
    }
    for (int np = 1; np <= 64 && P > 0; ++np) {
        Plan q = from;
        q.chunk_p = int(chunk(P, np)), q.np = int((P + q.chunk_p - 1) / q.chunk_p);
        const double items = double(base) * q.np;
        const double t = std::max(1.0, std::ceil(items / places)) * tiles(q.chunk_p) * tile_us + slot_us * (q.np + q.os);
        if (t < best) best = t, p = q;
    }
    return p;
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
    launch_attention<true>(s, kv, b, x, tree, plan_tree, workspace, bytes, "attention_tree");
}

}  // namespace omg
