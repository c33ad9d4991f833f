// The dense product's kernels for bf16 operands.
#include "gemm_dense.h"

namespace lo {
LO_DENSE_LAUNCHERS(LO_BF16)
} // namespace lo
