// The norm block's kernels for bf16.
#include "norm_block.hpp"

namespace cchip {
namespace op {
CCHIP_NORM_BLOCK_LAUNCHERS(bf16)
}  // namespace op
}  // namespace cchip
