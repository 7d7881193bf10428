// Attention of drafted tokens, which see the rows before them and, of the
// sequence's new rows, those that their masks name: the kernels of
// shared_attention.h with MASKED.  Only tiles that hold new rows look at the
// masks (a word or two a lane, asked for a tile ahead).
#include "shared_attention.h"

namespace omg {

int64_t attention_tree_workspace(const PagedKv& kv, const PagedBatch& b, int heads) {
    check(kv, b, heads, "attention_tree");
    return part_bytes(plan(kv, b, heads), kv, b, heads);
}

void launch_attention_tree(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const SharedAttn& x,
                           const TreeMask& tree, void* workspace, size_t bytes) {
    if (!tree.mask || reinterpret_cast<uintptr_t>(tree.mask) % 4)
        fail(E_INVALID, "attention_tree: mask must be a 4-byte aligned device pointer");
    if (tree.words <= 0 || tree.words > (1 << 20)) fail(E_INVALID, "attention_tree: mask_ld must be 1 to 2^20 words");
    if (x.window > 0 && !tree.positions) fail(E_INVALID, "attention_tree: a window needs the tokens' positions");
    if (reinterpret_cast<uintptr_t>(tree.positions) % 4) fail(E_INVALID, "attention_tree: positions must be 4-byte aligned");
    launch_attention<true>(s, kv, b, x, tree, workspace, bytes, "attention_tree");
}

}  // namespace omg
