// Attention's backward kernels for bf16.
#include "attention_backward.hpp"

namespace cchip {
namespace op {
template void attend_back_launch<bf16>(const AttentionArgs &, hipStream_t);
}  // namespace op
}  // namespace cchip
