// Attention for drafted trees: fp16 queries, int8 keys and values (the kernel is pda_tree.h's).

#include "pda_tree.h"

namespace pda_tree {

const void* tree_kernel_q8(int width, int waves, bool exact) {
  return tree_kernel_for<false, true>(width, waves, exact);
}

}  // namespace pda_tree
