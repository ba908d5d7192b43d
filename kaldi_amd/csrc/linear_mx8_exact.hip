// The linear operator's kernels for 8-bit operands widened to bf16 (see linear_kernels.h).
#define AMLIKE_LINEAR_KERNELS
#include "linear_kernels.h"

namespace amlike {
template int LaunchLinear<kMx8Exact>(const LinearArgs &, hipStream_t);
}  // namespace amlike
