// Attention for drafted trees: bf16 (the kernel is pda_tree.h's).

#include "pda_tree.h"

namespace pda_tree {

const void* tree_kernel_bf16(int width, int waves, bool exact) {
  return tree_kernel_for<true, false>(width, waves, exact);
}

}  // namespace pda_tree
