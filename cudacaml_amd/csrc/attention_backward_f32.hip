// Attention's backward kernels for f32.
#include "attention_backward.hpp"

namespace cchip {
namespace op {
template void attend_back_launch<float>(const AttentionArgs &, hipStream_t);
}  // namespace op
}  // namespace cchip
