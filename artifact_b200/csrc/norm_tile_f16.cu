// The kernels of norm_tile.cuh for float16 matrices.
#include "norm_tile.cuh"

namespace rof {
const TileLauncher tile_launcher_f16 = launch_tile<__half>;
}  // namespace rof
