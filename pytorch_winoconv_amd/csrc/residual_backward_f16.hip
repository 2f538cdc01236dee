#include "residual_backward.inc"

namespace wc {
template int join_backward_of<half_t>(const JoinGradients&, void*);
}  // namespace wc
