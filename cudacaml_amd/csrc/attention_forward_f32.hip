// Attention's forward kernels for f32.
#include "attention_forward.hpp"

namespace cchip {
namespace op {
template void attend_launch<float>(const AttentionArgs &, int, hipStream_t);
}  // namespace op
}  // namespace cchip
