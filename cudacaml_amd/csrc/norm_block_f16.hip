// The norm block's kernels for f16.
#include "norm_block.hpp"

namespace cchip {
namespace op {
CCHIP_NORM_BLOCK_LAUNCHERS(f16)
}  // namespace op
}  // namespace cchip
