// The kernels of norm_tile.cuh for 32-bit matrices.
#include "norm_tile.cuh"

namespace rof {
const TileLauncher tile_launcher_f32 = launch_tile<float>;
}  // namespace rof
