// The norm block's kernels for f32.
#include "norm_block.hpp"

namespace cchip {
namespace op {
CCHIP_NORM_BLOCK_LAUNCHERS(float)
}  // namespace op
}  // namespace cchip
