// Attention's forward kernels for bf16.
#include "attention_forward.hpp"

namespace cchip {
namespace op {
template void attend_launch<bf16>(const AttentionArgs &, int, hipStream_t);
}  // namespace op
}  // namespace cchip
