// The 4-bit linear layer's kernels for f16 rows of x (mx_linear.hpp).
#include "mx_linear.hpp"

namespace mbrt {
template int launch_mx_linear<F16>(MxLinArgs& a, int align, hipStream_t st);
}  // namespace mbrt
