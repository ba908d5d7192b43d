// The linear operator's kernels for bf16 operands (see linear_kernels.h).
#define AMLIKE_LINEAR_KERNELS
#include "linear_kernels.h"

namespace amlike {
template int LaunchLinear<AMLIKE_BF16>(const LinearArgs &, hipStream_t);
}  // namespace amlike
