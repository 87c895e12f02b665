// The linear layer's kernels for f16 operands (linear.hpp).
#include "linear.hpp"

namespace mbrt {
template int launch_linear<F16>(LinArgs& a, int align, hipStream_t st);
}  // namespace mbrt
