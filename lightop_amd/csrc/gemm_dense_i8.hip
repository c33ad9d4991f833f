// The dense product's kernels for int8 operands.
#include "gemm_dense.h"

namespace lo {
LO_DENSE_LAUNCHERS(LO_I8)
} // namespace lo
