#include "residual_backward.inc"

namespace wc {
template int join_backward_of<float>(const JoinGradients&, void*);
}  // namespace wc
