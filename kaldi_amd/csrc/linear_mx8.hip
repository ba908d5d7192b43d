// The linear operator's kernels for 8-bit operands (see linear_kernels.h).
#define AMLIKE_LINEAR_KERNELS
#include "linear_kernels.h"

namespace amlike {
template int LaunchLinear<AMLIKE_MX8>(const LinearArgs &, hipStream_t);
}  // namespace amlike
