// The kernels of norm_kernels.cuh for float16 matrices.
#include "norm_kernels.cuh"

namespace rof {
const NormLaunchers norm_launchers_f16 = launchers<__half>();
}  // namespace rof
