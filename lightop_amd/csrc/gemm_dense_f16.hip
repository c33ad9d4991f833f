// The dense product's kernels for fp16 operands.
#include "gemm_dense.h"

namespace lo {
LO_DENSE_LAUNCHERS(LO_F16)
} // namespace lo
