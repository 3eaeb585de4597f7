// The kernels of norm_kernels.cuh for 32-bit matrices.
#include "norm_kernels.cuh"

namespace rof {
const NormLaunchers norm_launchers_f32 = launchers<float>();
}  // namespace rof
