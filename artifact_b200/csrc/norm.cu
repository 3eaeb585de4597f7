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
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rof_internal.h"

namespace rof {
namespace {

// ---- types --------------------------------------------------------------------------------------
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// a weight or bias vector: 32-bit, or of the matrix's own type
template <class T>
struct Vector {
  const void* p;
  int f32;
  __device__ __forceinline__ float at(int i) const {
    return f32 ? __ldg(reinterpret_cast<const float*>(p) + i) : to_float(reinterpret_cast<const T*>(p)[i]);
  }
};

template <class T>
__device__ __forceinline__ void put(void* p, int f32, int i, float v) {
  if (f32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<T*>(p)[i] = from_float<T>(v);
}

// ---- generator ----------------------------------------------------------------------------------
struct Drop {
  uint32_t on;         // 0: no element is dropped
  uint32_t last;       // words up to this one are dropped
  float scale;         // 1 / (1 - p)
  uint32_t k0, k1;     // key
  uint64_t step;
  const int64_t* step_dev;   // added to `step` when the kernel runs
  int64_t first;       // index of the matrix's first element in the whole one
};

__device__ __forceinline__ uint4 philox7(uint64_t group, uint64_t step, uint32_t k0, uint32_t k1) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint64_t step_of(const Drop& d) {
  return d.on && d.step_dev != nullptr ? d.step + (uint64_t)*d.step_dev : d.step;
}

__device__ __forceinline__ bool kept(const Drop& d, uint64_t step, int64_t e) {
  const uint4 w = philox7((uint64_t)e >> 2, step, d.k0, d.k1);
  const uint32_t r = (e & 2) ? ((e & 1) ? w.w : w.z) : ((e & 1) ? w.y : w.x);
  return r > d.last;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// relu(z) and its gradient keep a NaN, as torch's do
__device__ __forceinline__ float relu_of(float z) { return z <= 0.0f ? 0.0f : z; }

struct NormArgs {
  const void* x; int64_t ldx;
  const void* dy; int64_t lddy;
  void* out; int64_t ldo;
  const void* weight; const void* bias; int wf32;
  float2* stats;
  float* partial;
  void* dweight; void* dbias;
  int64_t rows; int dim; int slabs; int64_t slab_rows;
  float eps; int relu;
  Drop drop;
};

__device__ __forceinline__ float affine(float h, float w, float b) { return __fmaf_rn(h, w, b); }

template <class T>
__global__ void __launch_bounds__(256) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = ((int64_t)gridDim.x * blockDim.x) >> 5;
  const Vector<T> w{a.weight, a.wf32}, b{a.bias, a.wf32};
  const uint64_t step = step_of(a.drop);
  for (int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < a.rows; r += warps) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    T* y = reinterpret_cast<T*>(a.out) + r * a.ldo;
    float s = 0.0f;
    for (int c = lane; c < a.dim; c += 32) s += to_float(x[c]);
    float mean = warp_sum(s) / (float)a.dim;
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = lane; c < a.dim; c += 32) {
      const float d = to_float(x[c]) - mean;
      s1 += d;
      s2 = __fmaf_rn(d, d, s2);
    }
    const float off = warp_sum(s1) / (float)a.dim;
    const float var = fmaxf(__fmaf_rn(-off, off, warp_sum(s2) / (float)a.dim), 0.0f);
    mean += off;
    const float rstd = __frsqrt_rn(var + a.eps);
    if (lane == 0 && a.stats != nullptr) a.stats[r] = make_float2(mean, rstd);
    for (int c = lane; c < a.dim; c += 32) {
      const float h = (to_float(x[c]) - mean) * rstd;
      float z = affine(h, a.weight ? w.at(c) : 1.0f, a.bias ? b.at(c) : 0.0f);
      if (a.relu) z = relu_of(z);
      if (a.drop.on) z = kept(a.drop, step, a.drop.first + r * a.dim + c) ? z * a.drop.scale : 0.0f;
      y[c] = from_float<T>(z);
    }
  }
}

// dz of one element of a layer norm's output
template <class T>
__device__ __forceinline__ float norm_dz(const NormArgs& a, uint64_t step, int64_t r, int c, float dy, float h, float w, float b) {
  float dz = dy;
  if (a.drop.on) dz = kept(a.drop, step, a.drop.first + r * a.dim + c) ? dz * a.drop.scale : 0.0f;
  if (a.relu && affine(h, w, b) <= 0.0f) dz = 0.0f;
  return dz;
}

template <class T>
__global__ void __launch_bounds__(256) norm_backward_rows_kernel(const __grid_constant__ NormArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t warps = ((int64_t)gridDim.x * blockDim.x) >> 5;
  const Vector<T> wv{a.weight, a.wf32}, bv{a.bias, a.wf32};
  const uint64_t step = step_of(a.drop);
  for (int64_t r = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; r < a.rows; r += warps) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    const T* dy = reinterpret_cast<const T*>(a.dy) + r * a.lddy;
    T* dx = reinterpret_cast<T*>(a.out) + r * a.ldo;
    const float2 st = a.stats[r];
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = lane; c < a.dim; c += 32) {
      const float h = (to_float(x[c]) - st.x) * st.y, w = a.weight ? wv.at(c) : 1.0f;
      const float g = w * norm_dz<T>(a, step, r, c, to_float(dy[c]), h, w, a.bias ? bv.at(c) : 0.0f);
      s1 += g;
      s2 = __fmaf_rn(g, h, s2);
    }
    s1 = warp_sum(s1) / (float)a.dim;
    s2 = warp_sum(s2) / (float)a.dim;
    for (int c = lane; c < a.dim; c += 32) {
      const float h = (to_float(x[c]) - st.x) * st.y, w = a.weight ? wv.at(c) : 1.0f;
      const float g = w * norm_dz<T>(a, step, r, c, to_float(dy[c]), h, w, a.bias ? bv.at(c) : 0.0f);
      dx[c] = from_float<T>(st.y * (g - s1 - h * s2));
    }
  }
}

// partial[slab][0..1][dim]: sums over the slab's rows of dz h and dz; thread = column
template <class T>
__global__ void __launch_bounds__(128) norm_backward_columns_kernel(const __grid_constant__ NormArgs a) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.dim) return;
  const Vector<T> wv{a.weight, a.wf32}, bv{a.bias, a.wf32};
  const uint64_t step = step_of(a.drop);
  const float w = a.weight ? wv.at(c) : 1.0f, b = a.bias ? bv.at(c) : 0.0f;
  const int64_t r0 = (int64_t)blockIdx.y * a.slab_rows, r1 = min(a.rows, r0 + a.slab_rows);
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float2 st = a.stats[r];
    const float h = (to_float(reinterpret_cast<const T*>(a.x)[r * a.ldx + c]) - st.x) * st.y;
    const float dz = norm_dz<T>(a, step, r, c, to_float(reinterpret_cast<const T*>(a.dy)[r * a.lddy + c]), h, w, b);
    s1 = __fmaf_rn(dz, h, s1);
    s2 += dz;
  }
  a.partial[((int64_t)blockIdx.y * 2 + 0) * a.dim + c] = s1;
  a.partial[((int64_t)blockIdx.y * 2 + 1) * a.dim + c] = s2;
}

// adds the slabs in order
template <class T>
__global__ void __launch_bounds__(128) join_columns_kernel(const float* partial, int slabs, int dim, void* first, void* second, int f32) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= dim) return;
  float s1 = 0.0f, s2 = 0.0f;
  for (int k = 0; k < slabs; ++k) {
    s1 += partial[((int64_t)k * 2 + 0) * dim + c];
    s2 += partial[((int64_t)k * 2 + 1) * dim + c];
  }
  if (first != nullptr) put<T>(first, f32, c, s1);
  if (second != nullptr) put<T>(second, f32, c, s2);
}

struct DropArgs {
  const void* x; int64_t ldx;      // forward: the input; backward: dy
  const void* y; int64_t ldy;      // backward with ReLU: the forward's output
  void* out; int64_t ldo;
  const void* bias; int bf32;
  float* partial; void* dbias;
  int64_t rows; int dim; int slabs; int64_t slab_rows;
  int relu;
  Drop drop;
};

template <class T>
__global__ void __launch_bounds__(256) dropout_forward_kernel(const __grid_constant__ DropArgs a) {
  const Vector<T> bv{a.bias, a.bf32};
  const uint64_t step = step_of(a.drop);
  const int64_t n = a.rows * a.dim, stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride) {
    const int64_t r = i / a.dim;
    const int c = (int)(i - r * a.dim);
    float z = to_float(reinterpret_cast<const T*>(a.x)[r * a.ldx + c]);
    if (a.bias) z += bv.at(c);
    if (a.relu) z = relu_of(z);
    if (a.drop.on) z = kept(a.drop, step, a.drop.first + i) ? z * a.drop.scale : 0.0f;
    reinterpret_cast<T*>(a.out)[r * a.ldo + c] = from_float<T>(z);
  }
}

// dz: with the ReLU the output says which elements were kept and positive
template <class T>
__device__ __forceinline__ float dropout_dz(const DropArgs& a, uint64_t step, int64_t r, int c) {
  float dz = to_float(reinterpret_cast<const T*>(a.x)[r * a.ldx + c]);
  if (a.relu) return to_float(reinterpret_cast<const T*>(a.y)[r * a.ldy + c]) <= 0.0f ? 0.0f : dz * a.drop.scale;
  if (a.drop.on) dz = kept(a.drop, step, a.drop.first + r * a.dim + c) ? dz * a.drop.scale : 0.0f;
  return dz;
}

template <class T>
__global__ void __launch_bounds__(256) dropout_backward_kernel(const __grid_constant__ DropArgs a) {
  const uint64_t step = step_of(a.drop);
  const int64_t n = a.rows * a.dim, stride = (int64_t)gridDim.x * blockDim.x;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride) {
    const int64_t r = i / a.dim;
    const int c = (int)(i - r * a.dim);
    reinterpret_cast<T*>(a.out)[r * a.ldo + c] = from_float<T>(dropout_dz<T>(a, step, r, c));
  }
}

template <class T>
__global__ void __launch_bounds__(128) dropout_columns_kernel(const __grid_constant__ DropArgs a) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= a.dim) return;
  const uint64_t step = step_of(a.drop);
  const int64_t r0 = (int64_t)blockIdx.y * a.slab_rows, r1 = min(a.rows, r0 + a.slab_rows);
  float s = 0.0f;
  for (int64_t r = r0; r < r1; ++r) s += dropout_dz<T>(a, step, r, c);
  a.partial[((int64_t)blockIdx.y * 2 + 0) * a.dim + c] = 0.0f;
  a.partial[((int64_t)blockIdx.y * 2 + 1) * a.dim + c] = s;
}

// ---- host ---------------------------------------------------------------------------------------
constexpr int kMaxSlabs = 1024;

int slabs_for(int64_t rows) { return (int)std::max<int64_t>(1, std::min<int64_t>(kMaxSlabs, (rows + 31) / 32)); }

int64_t column_workspace(int64_t rows, int dim) { return (int64_t)slabs_for(rows) * 2 * dim * 4; }

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
  *out = Drop{0, 0, 1.0f, 0, 0, 0, nullptr, 0};
  if (d == nullptr) return ROF_OK;
  if (!(d->p >= 0.0 && d->p <= 1.0)) return bad(who, "p is not in [0, 1]");
  if (d->first_row < 0 || (dim > 0 && d->first_row > INT64_MAX / 8 / dim)) return bad(who, "first_row out of range");
  if (!aligned(d->step_dev, 8)) return bad(who, "step_dev is not aligned to its element");
  const double border = std::nearbyint(d->p * 4294967296.0);
  if (border < 1.0) return ROF_OK;                 // nothing would be dropped
  out->on = 1;
  out->last = (uint32_t)((uint64_t)border - 1);
  out->scale = d->p < 1.0 ? (float)(1.0 / (1.0 - d->p)) : 0.0f;
  out->k0 = (uint32_t)d->seed;
  out->k1 = (uint32_t)(d->seed >> 32);
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

template <class F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case ROF_DTYPE_F32: f(float{}); break;
    case ROF_DTYPE_BF16: f(__nv_bfloat16{}); break;
    default: f(__half{}); break;
  }
  return ROF_OK;
}

int grid_for(int64_t threads) { return (int)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 148 * 8)); }

int launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? ROF_OK : cuda_fail(e, who);
}

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
  by_type(dtype, [&](auto t) {
    norm_forward_kernel<decltype(t)><<<grid_for(rows * 32), 256, 0, (cudaStream_t)stream>>>(a);
  });
  return launched(who);
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
  a.partial = reinterpret_cast<float*>(workspace); a.rows = rows; a.dim = dim; a.relu = relu != 0;
  a.slabs = slabs_for(rows); a.slab_rows = (rows + a.slabs - 1) / a.slabs;
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (dx != nullptr && rows > 0) norm_backward_rows_kernel<T><<<grid_for(rows * 32), 256, 0, stream>>>(a);
    if (columns) {
      norm_backward_columns_kernel<T><<<dim3((dim + 127) / 128, a.slabs), 128, 0, stream>>>(a);
      join_columns_kernel<T><<<(dim + 127) / 128, 128, 0, stream>>>(a.partial, a.slabs, dim, dweight, dbias, a.wf32);
    }
  });
  return launched(who);
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
  by_type(dtype, [&](auto t) {
    dropout_forward_kernel<decltype(t)><<<grid_for(rows * dim), 256, 0, (cudaStream_t)stream>>>(a);
  });
  return launched(who);
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
  a.x = dy; a.ldx = lddy; a.y = y; a.ldy = ldy; a.out = dx; a.ldo = lddx; a.bf32 = vdtype == ROF_DTYPE_F32;
  a.partial = reinterpret_cast<float*>(workspace); a.rows = rows; a.dim = dim; a.relu = relu != 0;
  a.slabs = slabs_for(rows); a.slab_rows = (rows + a.slabs - 1) / a.slabs;
  by_type(dtype, [&](auto t) {
    using T = decltype(t);
    if (dx != nullptr && rows > 0) dropout_backward_kernel<T><<<grid_for(rows * dim), 256, 0, stream>>>(a);
    if (dbias != nullptr) {
      dropout_columns_kernel<T><<<dim3((dim + 127) / 128, a.slabs), 128, 0, stream>>>(a);
      join_columns_kernel<T><<<(dim + 127) / 128, 128, 0, stream>>>(a.partial, a.slabs, dim, nullptr, dbias, a.bf32);
    }
  });
  return launched(who);
}

}  // extern "C"
