// Declarations shared by norm.cu (the C entry points) and the per-type translation units with the kernels.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>

namespace rof {

// the kernels' form of a rof_dropout
struct Drop {
  uint32_t on;         // 0: no element is dropped (scale is 1)
  uint32_t last;       // words up to this one are dropped
  float scale;         // 1 / (1 - p)
  uint32_t key[14];    // of the seven rounds: two words each
  uint64_t step;
  const int64_t* step_dev;   // added to `step` when the kernel runs
  int64_t first;       // index of the matrix's first element in the whole one
};

struct NormArgs {
  const void* x; int64_t ldx;
  const void* dy; int64_t lddy;
  void* out; int64_t ldo;             // y, or dx (null: not wanted)
  const void* weight; const void* bias; int wf32;
  float2* stats;                      // mean and rstd of every row
  float* partial;                     // [blocks][2][dim] (null: no column sums)
  void* dweight; void* dbias;
  int64_t rows; int dim;
  float eps; int relu;
  Drop drop;
};

struct DropArgs {
  const void* x; int64_t ldx;         // forward: the input; backward: dy
  const void* y; int64_t ldy;         // backward with ReLU: the forward's output
  void* out; int64_t ldo;             // y, or dx (null: not wanted)
  const void* bias; int bf32;
  float* partial; void* dbias;        // [blocks][dim] (null: no column sums)
  int64_t rows; int dim;
  int relu;
  int lanes;                          // set by the launcher: threads that cover a tile of a row
  Drop drop;
};

// The backward kernels leave one set of column sums per block.  At most this many blocks, a multiple of 8 (the rows of a block
// keep their distance to the 16-byte boundaries), and at most 64 MB of sums unless the rows are very wide.
constexpr int kMaxColumnBlocks = 1184;
inline int column_blocks_cap(int64_t rows, int dim) {
  const int64_t fit = std::max<int64_t>(144, (64 << 20) / (8 * (int64_t)std::max(dim, 1)));
  const int64_t cap = std::min<int64_t>(kMaxColumnBlocks, fit) / 8 * 8;
  return (int)std::min<int64_t>(cap, (std::max<int64_t>(rows, 1) + 7) / 8 * 8);
}

// Whether a 16-byte vector of `vec` elements whose first is in column c of row r ends in the matrix.  One that passes the end of its row
// reaches up to vec - 1 elements further: into rows of one column and more, of which that many follow.
__host__ __device__ inline bool ends_in_matrix(int64_t r, int64_t rows, int c, int dim, int vec) { return c + vec <= dim || r < rows - vec; }

// The tile kernels (norm_tile.cuh).
enum TileMode { kNormForward, kNormForwardHidden, kNormBackward, kNormBackwardHidden, kDropForward, kDropBackward };

constexpr int kTileMaxColumns = 511;

struct RowRunArgs {
  const void* a;            // x, or a dropout's dy
  const void* b;            // a norm's dy, or the dropout's output (null: not read)
  void* out;
  const void* weight; const void* bias; int f32;
  float2* stats;
  float* partial;           // [blocks][2 (norm) or 1][dim]
  int64_t rows; int dim;
  float eps; int relu;
  Drop drop;
};

struct NormLaunchers {
  cudaError_t (*norm_forward)(const NormArgs&, cudaStream_t);
  cudaError_t (*norm_backward)(const NormArgs&, cudaStream_t);
  cudaError_t (*dropout_forward)(const DropArgs&, cudaStream_t);
  cudaError_t (*dropout_backward)(const DropArgs&, cudaStream_t);
};
using TileLauncher = cudaError_t (*)(const RowRunArgs&, int mode, cudaStream_t, int* blocks);
extern const TileLauncher tile_launcher_f32, tile_launcher_bf16, tile_launcher_f16;
extern const NormLaunchers norm_launchers_f32, norm_launchers_bf16, norm_launchers_f16;

}  // namespace rof
