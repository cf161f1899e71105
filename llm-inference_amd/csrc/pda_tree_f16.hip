// Attention for drafted trees: fp16 (the kernel is pda_tree.h's).

#include "pda_tree.h"

namespace pda_tree {

const void* tree_kernel_f16(int width, int waves, bool exact) {
  return tree_kernel_for<false, false>(width, waves, exact);
}

}  // namespace pda_tree
