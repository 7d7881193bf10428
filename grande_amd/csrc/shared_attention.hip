// Attention over a shared prefix and every sequence's own rows, each token
// seeing its sequence up to itself.
#include "shared_attention.h"

namespace omg {

int64_t attention_shared_workspace(const PagedKv& kv, const PagedBatch& b, int heads) {
    check(kv, b, heads, "attention_shared");
    return part_bytes(plan(kv, b, heads), kv, b, heads);
}

void launch_attention_shared(hipStream_t s, const PagedKv& kv, const PagedBatch& b, const SharedAttn& x,
                             void* workspace, size_t bytes) {
    launch_attention<false>(s, kv, b, x, TreeMask{}, plan, workspace, bytes, "attention_shared");
}

}  // namespace omg
