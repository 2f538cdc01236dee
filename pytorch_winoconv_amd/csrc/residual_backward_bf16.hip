#include "residual_backward.inc"

namespace wc {
template int join_backward_of<bf16_t>(const JoinGradients&, void*);
}  // namespace wc
