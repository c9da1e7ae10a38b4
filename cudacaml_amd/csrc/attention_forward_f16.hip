// Attention's forward kernels for f16.
#include "attention_forward.hpp"

namespace cchip {
namespace op {
template void attend_launch<f16>(const AttentionArgs &, int, hipStream_t);
}  // namespace op
}  // namespace cchip
