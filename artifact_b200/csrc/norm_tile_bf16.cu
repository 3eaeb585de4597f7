// The kernels of norm_tile.cuh for bfloat16 matrices.
#include "norm_tile.cuh"

namespace rof {
const TileLauncher tile_launcher_bf16 = launch_tile<__nv_bfloat16>;
}  // namespace rof
