// The kernels of norm_kernels.cuh for bfloat16 matrices.
#include "norm_kernels.cuh"

namespace rof {
const NormLaunchers norm_launchers_bf16 = launchers<__nv_bfloat16>();
}  // namespace rof
