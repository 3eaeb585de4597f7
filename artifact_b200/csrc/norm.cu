// The operators between two graph layers: layer norm, dropout from a counter-based generator, and both
// in one pass with the ReLU between them (bias add and ReLU in front of dropout without a norm).
//
// Layer norm of a row of D values:
//     mean = sum x / D, rstd = 1 / sqrt(sum (x - mean)^2 / D + eps), h = (x - mean) rstd, z = h w + b
// and back, with g = dz w:
//     dx = rstd (g - sum g / D - h sum (g h) / D),  dw = sum over rows of dz h,  db = sum over rows of dz.
// Dropout keeps element e = row * D + column of the whole matrix where its random word is not below
// p * 2^32 and scales it by 1 / (1 - p); the word is word e % 4 of Philox4x32 (seven rounds; Salmon et al., "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011, where seven is the fewest that pass its test battery) at
// counter (e / 4, step) under the key `seed`.  The backward pass computes the words again.
//
// Everything is held in 32 bits between the load and the one rounding at the store.
#include <cmath>
#include <cstdint>
#include <string>

#include "norm.h"
#include "rof_internal.h"

namespace rof {
namespace {

int64_t column_workspace(int64_t rows, int dim) { return (int64_t)column_blocks_cap(rows, dim) * 2 * dim * 4; }

int bad(const char* who, const char* what) {
  set_error(std::string(who) + ": " + what);
  return ROF_ERR_BAD_ARGUMENT;
}

int element_bytes(int dtype) { return dtype == ROF_DTYPE_F32 ? 4 : 2; }

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

// the sizes all entry points share
int check_sizes(const char* who, int dtype, int vdtype, int64_t rows, int dim) {
  if (dtype < 0 || dtype > ROF_DTYPE_F16) return bad(who, "unknown element type");
  if (vdtype != ROF_DTYPE_F32 && vdtype != dtype) return bad(who, "vectors are 32-bit or of the matrix's type");
  if (rows < 0 || dim < 0) return bad(who, "negative size");
  if (dim > (1 << 30)) return bad(who, "rows of more than 2^30 columns");
  if (dim > 0 && rows > INT64_MAX / 8 / dim) return bad(who, "too many elements");
  return ROF_OK;
}

int check_matrix(const char* who, const char* name, int dtype, const void* p, int64_t ld, int64_t rows, int dim) {
  if (p == nullptr) return bad(who, (std::string("null ") + name).c_str());
  if (!aligned(p, element_bytes(dtype))) return bad(who, (std::string(name) + " is not aligned to its elements").c_str());
  if (rows > 1 && (ld < dim || ld > INT64_MAX / 8 / rows)) return bad(who, (std::string("row stride of ") + name + " out of range").c_str());
  return ROF_OK;
}

// the kernels' form of a rof_dropout
int read_drop(const char* who, const rof_dropout* d, int64_t rows, int dim, Drop* out) {
  *out = Drop{};
  out->scale = 1.0f;
  if (d == nullptr) return ROF_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return bad(who, "p is not in [0, 1]");
  if (d->first_row < 0 || (dim > 0 && d->first_row > INT64_MAX / 8 / dim)) return bad(who, "first_row out of range");
  if (!aligned(d->step_dev, 8)) return bad(who, "step_dev is not aligned to its element");
  const double border = std::nearbyint(d->p * 4294967296.0);
  if (border < 1.0) return ROF_OK;                 // nothing would be dropped
  out->on = 1;
  out->last = (uint32_t)((uint64_t)border - 1);
  out->scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.0f;
  for (int i = 0; i < 7; ++i) {                    // the key moves on by these two constants from round to round
    out->key[2 * i] = (uint32_t)d->seed + (uint32_t)i * 0x9E3779B9u;
    out->key[2 * i + 1] = (uint32_t)(d->seed >> 32) + (uint32_t)i * 0xBB67AE85u;
  }
  out->step = d->step;
  out->step_dev = d->step_dev;
  out->first = d->first_row * dim;
  return ROF_OK;
}

int check_workspace(const char* who, const void* ws, int64_t have, int64_t need) {
  if (ws != nullptr && have >= need && aligned(ws, 256)) return ROF_OK;
  set_error(std::string(who) + ": workspace missing, not 256-byte aligned, or smaller than rof_layer_norm_workspace_bytes()");
  return ROF_ERR_WORKSPACE;
}

const NormLaunchers& launchers_of(int dtype) {
  return dtype == ROF_DTYPE_F32 ? norm_launchers_f32 : dtype == ROF_DTYPE_BF16 ? norm_launchers_bf16 : norm_launchers_f16;
}

int status(const char* who, cudaError_t e) { return e == cudaSuccess ? ROF_OK : cuda_fail(e, who); }

}  // namespace
}  // namespace rof

using namespace rof;

extern "C" {

int64_t rof_layer_norm_workspace_bytes(int64_t rows, int dim) {
  if (rows < 0 || dim < 0) return -1;
  return column_workspace(rows, dim);
}

int rof_layer_norm_forward(int dtype, const void* x, int64_t ldx, int64_t rows, int dim, int vdtype, const void* weight,
                           const void* bias, float eps, int relu, const rof_dropout* drop, void* y, int64_t ldy,
                           float* stats, void* stream) {
  static const char who[] = "rof_layer_norm_forward";
  NormArgs a{};
  int rc = check_sizes(who, dtype, vdtype, rows, dim);
  if (rc == ROF_OK) rc = read_drop(who, drop, rows, dim, &a.drop);
  if (rc != ROF_OK) return rc;
  if (!(eps >= 0.0f)) return bad(who, "eps is negative or not a number");
  if (rows == 0 || dim == 0) return ROF_OK;
  if ((rc = check_matrix(who, "x", dtype, x, ldx, rows, dim)) || (rc = check_matrix(who, "y", dtype, y, ldy, rows, dim))) return rc;
  if (!aligned(weight, element_bytes(vdtype)) || !aligned(bias, element_bytes(vdtype)) || !aligned(stats, 8)) return bad(who, "misaligned vector");
  a.x = x; a.ldx = ldx; a.out = y; a.ldo = ldy; a.weight = weight; a.bias = bias; a.wf32 = vdtype == ROF_DTYPE_F32;
  a.stats = reinterpret_cast<float2*>(stats);
  a.rows = rows; a.dim = dim; a.eps = eps; a.relu = relu != 0;
  return status(who, launchers_of(dtype).norm_forward(a, (cudaStream_t)stream));
}

int rof_layer_norm_backward(int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, int64_t rows, int dim,
                            int vdtype, const void* weight, const void* bias, const float* stats, int relu,
                            const rof_dropout* drop, void* dx, int64_t lddx, void* dweight, void* dbias,
                            void* workspace, int64_t workspace_bytes, void* stream_) {
  static const char who[] = "rof_layer_norm_backward";
  cudaStream_t stream = (cudaStream_t)stream_;
  NormArgs a{};
  int rc = check_sizes(who, dtype, vdtype, rows, dim);
  if (rc == ROF_OK) rc = read_drop(who, drop, rows, dim, &a.drop);
  if (rc != ROF_OK) return rc;
  if (dim == 0 || (dx == nullptr && dweight == nullptr && dbias == nullptr)) return ROF_OK;
  const bool columns = dweight != nullptr || dbias != nullptr;
  if (!aligned(weight, element_bytes(vdtype)) || !aligned(bias, element_bytes(vdtype)) || !aligned(stats, 8) ||
      !aligned(dweight, element_bytes(vdtype)) || !aligned(dbias, element_bytes(vdtype))) return bad(who, "misaligned vector");
  if (rows > 0) {
    if ((rc = check_matrix(who, "x", dtype, x, ldx, rows, dim)) || (rc = check_matrix(who, "dy", dtype, dy, lddy, rows, dim)) ||
        (dx != nullptr && (rc = check_matrix(who, "dx", dtype, dx, lddx, rows, dim)))) return rc;
    if (stats == nullptr) return bad(who, "null stats");
  }
  if (columns && (rc = check_workspace(who, workspace, workspace_bytes, column_workspace(rows, dim)))) return rc;
  a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.out = dx; a.ldo = lddx; a.weight = weight; a.bias = bias;
  a.wf32 = vdtype == ROF_DTYPE_F32; a.stats = const_cast<float2*>(reinterpret_cast<const float2*>(stats));
  a.partial = columns ? reinterpret_cast<float*>(workspace) : nullptr; a.dweight = dweight; a.dbias = dbias;
  a.rows = rows; a.dim = dim; a.relu = relu != 0;
  return status(who, launchers_of(dtype).norm_backward(a, stream));
}

int rof_dropout_forward(int dtype, const void* x, int64_t ldx, int64_t rows, int dim, int vdtype, const void* bias, int relu,
                        const rof_dropout* drop, void* y, int64_t ldy, void* stream) {
  static const char who[] = "rof_dropout_forward";
  DropArgs a{};
  int rc = check_sizes(who, dtype, vdtype, rows, dim);
  if (rc == ROF_OK) rc = read_drop(who, drop, rows, dim, &a.drop);
  if (rc != ROF_OK) return rc;
  if (rows == 0 || dim == 0) return ROF_OK;
  if ((rc = check_matrix(who, "x", dtype, x, ldx, rows, dim)) || (rc = check_matrix(who, "y", dtype, y, ldy, rows, dim))) return rc;
  if (!aligned(bias, element_bytes(vdtype))) return bad(who, "misaligned vector");
  a.x = x; a.ldx = ldx; a.out = y; a.ldo = ldy; a.bias = bias; a.bf32 = vdtype == ROF_DTYPE_F32;
  a.rows = rows; a.dim = dim; a.relu = relu != 0;
  return status(who, launchers_of(dtype).dropout_forward(a, (cudaStream_t)stream));
}

int rof_dropout_backward(int dtype, const void* dy, int64_t lddy, const void* y, int64_t ldy, int64_t rows, int dim, int vdtype,
                         int relu, const rof_dropout* drop, void* dx, int64_t lddx, void* dbias, void* workspace,
                         int64_t workspace_bytes, void* stream_) {
  static const char who[] = "rof_dropout_backward";
  cudaStream_t stream = (cudaStream_t)stream_;
  DropArgs a{};
  int rc = check_sizes(who, dtype, vdtype, rows, dim);
  if (rc == ROF_OK) rc = read_drop(who, drop, rows, dim, &a.drop);
  if (rc != ROF_OK) return rc;
  if (dim == 0 || (dx == nullptr && dbias == nullptr)) return ROF_OK;
  if (!aligned(dbias, element_bytes(vdtype))) return bad(who, "misaligned vector");
  if (rows > 0) {
    if ((rc = check_matrix(who, "dy", dtype, dy, lddy, rows, dim)) ||
        (relu && (rc = check_matrix(who, "y", dtype, y, ldy, rows, dim))) ||
        (dx != nullptr && (rc = check_matrix(who, "dx", dtype, dx, lddx, rows, dim)))) return rc;
  }
  if (dbias != nullptr && (rc = check_workspace(who, workspace, workspace_bytes, column_workspace(rows, dim)))) return rc;
  a.x = dy; a.ldx = lddy; a.y = relu ? y : nullptr; a.ldy = ldy; a.out = dx; a.ldo = lddx; a.bf32 = vdtype == ROF_DTYPE_F32;
  a.partial = dbias != nullptr ? reinterpret_cast<float*>(workspace) : nullptr; a.dbias = dbias;
  a.rows = rows; a.dim = dim; a.relu = relu != 0;
  return status(who, launchers_of(dtype).dropout_backward(a, stream));
}

}  // extern "C"
