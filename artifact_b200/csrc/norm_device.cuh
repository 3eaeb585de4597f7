// Device code that the kernels of layer norm and dropout share: types, 16-byte vectors, asynchronous copies, the
// generator, sums over a group of threads.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cfloat>
#include <initializer_list>
#include <type_traits>

#include "norm.h"

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

template <class T> constexpr int kVec = 16 / (int)sizeof(T);

// a weight or bias vector: 32-bit, or of the matrix's own type
template <class T>
__device__ __forceinline__ float vector_at(const void* p, int f32, int i) {
  return f32 ? __ldg(reinterpret_cast<const float*>(p) + i) : to_float(reinterpret_cast<const T*>(p)[i]);
}

template <class T>
__device__ __forceinline__ void vector_put(void* p, int f32, int i, float v) {
  if (f32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<T*>(p)[i] = from_float<T>(v);
}

template <class T>
union Pack {
  uint4 raw;
  T v[kVec<T>];
  __device__ Pack() {}
};

// Columns [c, c + VEC) of row r, c + VEC > 0.  Partial vectors hold what the 16 bytes hold, the neighbouring
// row's elements or what precedes the matrix in its allocation; behind the end of the matrix nothing is read.
template <class T, bool EDGE>
__device__ __forceinline__ void load_vec(Pack<T>& out, const T* row, int c, int dim, int64_t r, int64_t rows) {
  if (!EDGE || ends_in_matrix(r, rows, c, dim, kVec<T>)) {
    out.raw = *reinterpret_cast<const uint4*>(row + c);
  } else {
#pragma unroll
    for (int t = 0; t < kVec<T>; ++t) out.v[t] = (unsigned)(c + t) < (unsigned)dim ? row[c + t] : from_float<T>(0.0f);
  }
}

__device__ __forceinline__ void pack_two(float* p, float2 v) { *reinterpret_cast<float2*>(p) = v; }
__device__ __forceinline__ void pack_two(__nv_bfloat16* p, float2 v) { *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v); }
__device__ __forceinline__ void pack_two(__half* p, float2 v) { *reinterpret_cast<__half2*>(p) = __float22half2_rn(v); }

// ---- asynchronous copies -------------------------------------------------------------------------
// 16 bytes from global to shared memory, the last 16 - bytes of them zero and not read
__device__ __forceinline__ void copy_async(uint4* to, const void* from, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void pair_copy(float* to, const float* from) { *reinterpret_cast<float2*>(to) = *reinterpret_cast<const float2*>(from); }
__device__ __forceinline__ void pair_copy(__nv_bfloat16* to, const __nv_bfloat16* from) { *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from); }
__device__ __forceinline__ void pair_copy(__half* to, const __half* from) { *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from); }

__device__ __forceinline__ void four_copy(float* to, const float* from) { *reinterpret_cast<float4*>(to) = *reinterpret_cast<const float4*>(from); }
template <class T>
__device__ __forceinline__ void four_copy(T* to, const T* from) { *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from); }

// A thread's own ring of S slots in shared memory for the C vectors of its next rows.  Every thread reads only what it copied
// itself, so the ring needs no barrier: it is an extension of the registers that keeps (S - 1) C vectors a thread in
// flight whatever the compiler does with the loads.  A slot is refilled one row after it was read.  Vectors that lie behind the
// row are cleared once and never copied.
//
// The kernels are short of instruction slots as much as of bandwidth in 16 bits, so addresses run along: `from` points to column c0 of the
// next row to fetch, and only additions remain in the loop.
template <class T, int L, int C, int S, bool EDGE>
struct Ring {
  char* mine;                // this thread's first vector of slot 0
  const char* from;
  int64_t row_bytes;         // from one row of the group to its next
  int left, advance;         // bytes from c0 to the end of the row; between two of the thread's vectors
  int threads;               // of the block
  __device__ __forceinline__ Ring(uint4* smem, int part, const void* base, int64_t ld, int64_t first, int64_t stride, int c0, int lanes, int dim) {
    threads = L == 0 ? (int)blockDim.x : 256;
    mine = reinterpret_cast<char*>(smem + (size_t)part * S * C * threads + threadIdx.x);
    from = reinterpret_cast<const char*>(reinterpret_cast<const T*>(base) + first * ld + c0);
    row_bytes = stride * ld * (int64_t)sizeof(T);
    left = (dim - c0) * (int)sizeof(T);
    advance = 16 * lanes;
#pragma unroll
    for (int i = 0; i < S * C; ++i)
      if (i % C * advance >= left) *reinterpret_cast<uint4*>(mine + i * threads * 16) = make_uint4(0, 0, 0, 0);
  }
  // The next row into the slot at byte `at`.  What lies behind it is zero.  In front of it (c0 < 0) the vector holds what
  // the 16 bytes hold: the end of the row before, or what precedes the matrix in its allocation; read() clears it.
  __device__ __forceinline__ void fetch(int at) {
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (k * advance < left)
        copy_async(reinterpret_cast<uint4*>(mine + at + k * threads * 16), from + k * advance, EDGE ? min(16, left - k * advance) : 16);
    from += row_bytes;
  }
  __device__ __forceinline__ void read(int at, Pack<T> (&out)[C], int c0) const {
#pragma unroll
    for (int k = 0; k < C; ++k) out[k].raw = *reinterpret_cast<const uint4*>(mine + at + k * threads * 16);
    if (EDGE && c0 < 0) {
#pragma unroll
      for (int t = 0; t < kVec<T>; ++t)
        if (c0 + t < 0) out[0].v[t] = from_float<T>(0.0f);
    }
  }
  __device__ __forceinline__ int slot_bytes() const { return C * threads * 16; }
  // Stores a row whose output lies differently against the 16-byte boundaries than its input: the group's vectors go into the
  // slot that was just read, and out of it element by element (W at a time), neighbours by neighbouring lanes.
  template <int W, class G>
  __device__ __forceinline__ void store_through(int at, const float2 (&v)[C][kVec<T> / 2], const G& g, T* out, int shift, int dim) const {
    constexpr int V = kVec<T>;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      Pack<T> p;
#pragma unroll
      for (int t = 0; t < V / 2; ++t) pack_two(&p.v[2 * t], v[k][t]);
      if (k * advance < left) *reinterpret_cast<uint4*>(mine + at + k * threads * 16) = p.raw;   // (the others stay cleared)
    }
    g.sync();
    // vector i of the row is vector i % lanes of the group's slice number i / lanes
    const T* slot = reinterpret_cast<const T*>(mine + at - g.lane * 16);
#pragma unroll
    for (int j = 0; j < C * V / W; ++j) {
      const int c = (g.lane + j * g.lanes) * W, e = c + shift, i = e / V;
      if (c < dim) {
        int k = 0;
#pragma unroll
        for (int q = 1; q < C; ++q) k += i >= q * g.lanes;
        const T* from = slot + (k * threads + (i - k * g.lanes)) * V + e % V;
        if constexpr (W == 2) pair_copy(out + c, from);
        else out[c] = *from;
      }
    }
    g.sync();
  }
};

// 1 / sqrt(v): the approximation and one Newton step, within a unit in the last place; 0 of infinity, whose product with the
// approximation would be a NaN
__device__ __forceinline__ float rsqrt_of(float v) {
  const float r = rsqrtf(v);
  return __fmaf_rn(0.5f * r, __fmaf_rn(-(fminf(v, FLT_MAX) * r), r, 1.0f), r);
}

// The variance from a row's mean square deviation from a first mean that is `off` from the mean.  Where the squares pass the range of
// 32 bits it is infinite: the row then has rstd 0 and becomes its bias.  (`square` is no less than off^2, so an `off` whose square is out of
// range stands beside an infinite one: it may be any smaller number.)
__device__ __forceinline__ float variance_of(float square, float off) {
  off = fminf(fabsf(off), 0x1.fffffep63f);
  return fmaxf(__fmaf_rn(-off, off, square), 0.0f);
}

// Two elements at a time: the f32x2 instructions of sm_100, each half rounded like the scalar one.
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// ---- generator ----------------------------------------------------------------------------------
__device__ __forceinline__ uint4 philox7(uint64_t group, uint64_t step, const uint32_t (&key)[14]) {
  uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t a = (uint64_t)0xD2511F53u * c0, b = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ key[2 * r];
    c2 = (uint32_t)(a >> 32) ^ c3 ^ key[2 * r + 1];
    c1 = (uint32_t)b;
    c3 = (uint32_t)a;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint64_t step_of(const Drop& d) {
  return d.on && d.step_dev != nullptr ? d.step + (uint64_t)*d.step_dev : d.step;
}

__device__ __forceinline__ uint32_t word(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

__device__ __forceinline__ bool kept(const Drop& d, uint64_t step, int64_t e) {
  return word(philox7((uint64_t)e >> 2, step, d.key), (int)(e & 3)) > d.last;
}

// The words of C runs of N elements: w[k N + t] is that of element e + k advance + t; N and advance are multiples of four.  One
// Philox call gives the words of four elements that start at a multiple of four.  Elsewhere (EDGE only: rows with a stride or an
// offset of their own) the elements lie in N / 4 + 1 such groups.  (No branch between the calls: seven rounds are one long
// chain of dependent instructions, and only other calls fill it.)
template <int C, int N, bool EDGE>
__device__ __forceinline__ void draw_words(const Drop& d, uint64_t step, int64_t e, int advance, uint32_t (&w)[C * N]) {
  const int sh = EDGE ? (int)(e & 3) : 0;
  if (!EDGE || sh == 0) {
#pragma unroll
    for (int i = 0; i < C * N / 4; ++i) {
      const uint4 g = philox7((uint64_t)(e >> 2) + (i / (N / 4) * (advance >> 2) + i % (N / 4)), step, d.key);
      w[4 * i] = g.x;
      w[4 * i + 1] = g.y;
      w[4 * i + 2] = g.z;
      w[4 * i + 3] = g.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < C; ++k) {
      uint4 a = philox7((uint64_t)((e + k * advance) >> 2), step, d.key);
#pragma unroll
      for (int q = 0; q < N / 4; ++q) {
        const uint4 b = philox7((uint64_t)((e + k * advance) >> 2) + q + 1, step, d.key);
        uint32_t* o = &w[k * N + 4 * q];
        o[0] = sh == 1 ? a.y : sh == 2 ? a.z : a.w;
        o[1] = sh == 1 ? a.z : sh == 2 ? a.w : b.x;
        o[2] = sh == 1 ? a.w : sh == 2 ? b.x : b.y;
        o[3] = sh == 1 ? b.x : sh == 2 ? b.y : b.z;
        a = b;
      }
    }
  }
}

// what stays of two elements with the words w[0] and w[1]
__device__ __forceinline__ float2 kept_of(const Drop& d, const uint32_t* w, float2 v, float dropped = 0.0f) {
  return make_float2(w[0] > d.last ? v.x : dropped, w[1] > d.last ? v.y : dropped);
}

// every element times f
template <int C, int H>
__device__ __forceinline__ void scale_elements(float2 (&v)[C][H], float f) {
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int t = 0; t < H; ++t) v[k][t] = __fmul2_rn(v[k][t], both(f));
}

// relu(z) and its gradient keep a NaN, as torch's do
__device__ __forceinline__ float relu_of(float z) {
  asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(z));
  return z;
}

// Behind a ReLU a dropout's backward pass asks the output which elements were kept and positive.  With a 32-bit bias a sum may be positive
// and still round to a zero of a 16-bit type.  That zero is stored with its sign set; every other zero is +0.  On the way the signs are
// the other way round, because the rounding then keeps them apart by itself: what is not positive or dropped is negative or -0
// (`scaled`: an exact zero is taken down by the least number there is), what is positive is +0 at least.  So two elements cost the ReLU
// as a maximum with -0, a comparison and an exclusive or (1000000x64 bf16: 67 us forward; choosing in
// 32 bits 84; without marks, the ReLU in 32 bits, 73).
constexpr float kLeast = 0x1p-149f;
template <class T, int C, int H>
__device__ __forceinline__ void scaled(float2 (&v)[C][H], float f, bool relu) {
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int t = 0; t < H; ++t) v[k][t] = __ffma2_rn(v[k][t], both(f), both(relu ? -kLeast : -0.0f));
}
template <class T>
__device__ __forceinline__ uint32_t relu_marked(uint32_t two) {
  const uint32_t none = 0x80008000u;
  uint32_t zeros;
  if constexpr (std::is_same<T, __half>::value) {
    asm("max.NaN.f16x2 %0, %0, %1;" : "+r"(two) : "r"(none));
    zeros = __heq2_mask(*reinterpret_cast<const __half2*>(&two), __half2{});
  } else {
    asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(two) : "r"(none));
    zeros = __heq2_mask(*reinterpret_cast<const __nv_bfloat162*>(&two), __nv_bfloat162{});
  }
  return two ^ (zeros & none);
}
template <class T>
__device__ __forceinline__ T relu_marked_one(T v) {
  const uint16_t one = (uint16_t)relu_marked<T>(*reinterpret_cast<const uint16_t*>(&v));
  return *reinterpret_cast<const T*>(&one);
}
template <class T>
__device__ __forceinline__ bool passed(T y) {
  if constexpr (sizeof(T) == 4) return __float_as_uint(y) != 0;
  else return *reinterpret_cast<const uint16_t*>(&y) != 0;
}
__device__ __forceinline__ float passed_of(float y, float v) { return __float_as_uint(y) != 0 ? v : 0.0f; }

__device__ __forceinline__ float affine(float h, float w, float b) { return __fmaf_rn(h, w, b); }

template <class T>
__device__ __forceinline__ void unpack(const Pack<T>& p, float2 (&v)[kVec<T> / 2]) {
#pragma unroll
  for (int t = 0; t < kVec<T> / 2; ++t) v[t] = make_float2(to_float(p.v[2 * t]), to_float(p.v[2 * t + 1]));
}

__device__ __forceinline__ float half_of(const float2& v, int i) { return i ? v.y : v.x; }

// `relu`: the 16-bit ReLU of relu_marked() on the way
template <class T, bool EDGE>
__device__ __forceinline__ void store_vec(T* row, int c, int dim, const float2 (&v)[kVec<T> / 2], bool relu = false) {
  Pack<T> p;
#pragma unroll
  for (int t = 0; t < kVec<T> / 2; ++t) pack_two(&p.v[2 * t], v[t]);
  if constexpr (sizeof(T) == 2) {
    if (relu) p.raw = make_uint4(relu_marked<T>(p.raw.x), relu_marked<T>(p.raw.y), relu_marked<T>(p.raw.z), relu_marked<T>(p.raw.w));
  }
  if (!EDGE || (c >= 0 && c + kVec<T> <= dim)) {
    *reinterpret_cast<uint4*>(row + c) = p.raw;
  } else {
#pragma unroll
    for (int t = 0; t < kVec<T>; ++t)
      if ((unsigned)(c + t) < (unsigned)dim) row[c + t] = p.v[t];
  }
}

// ---- groups -------------------------------------------------------------------------------------
// L = 4..32: lanes of a warp; L = 0: the block is the group
template <int L>
struct Group {
  int lane, lanes, index;      // index: of the group in the block
  unsigned mask;
  int64_t first, stride;       // rows of this group: first, first + stride, ...
  __device__ __forceinline__ Group() {
    if constexpr (L == 0) {
      lane = threadIdx.x;
      lanes = blockDim.x;
      index = 0;
      mask = 0xffffffffu;
      first = blockIdx.x;
      stride = gridDim.x;
    } else {
      lane = threadIdx.x % L;
      lanes = L;
      index = threadIdx.x / L;
      mask = L == 32 ? 0xffffffffu : ((1u << (L & 31)) - 1u) << ((threadIdx.x & 31) & ~(L - 1));
      first = (int64_t)blockIdx.x * (blockDim.x / L) + index;
      stride = (int64_t)gridDim.x * (blockDim.x / L);
    }
  }
  __device__ __forceinline__ void sync() const {
    if constexpr (L == 0) __syncthreads();
    else __syncwarp(mask);
  }
  // Sums over the group, the same in every lane, always added in the same order.  `buf`: two floats per warp, another one
  // for each of two sums that follow one another (L = 0 only).
  __device__ __forceinline__ float sum(float v, float* buf) const {
#pragma unroll
    for (int o = (L == 0 ? 32 : L) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(mask, v, o);
    if constexpr (L == 0) {
      const int warps = blockDim.x >> 5;
      if (warps > 1) {
        if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < warps ? buf[threadIdx.x & 31] : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)              // at most 16 warps
          if (o < warps) v += __shfl_xor_sync(mask, v, o);
        v = __shfl_sync(mask, v, 0);
      }
    }
    return v;
  }
  // two sums at once: the first exchange leaves one of them to each half of the group
  __device__ __forceinline__ float2 sum(float2 v, float* buf) const {
    constexpr int W = L == 0 ? 32 : L;
    const bool upper = threadIdx.x & (W / 2);
    const float other = __shfl_xor_sync(mask, upper ? v.x : v.y, W / 2);
    float mine = (upper ? v.y : v.x) + other;
#pragma unroll
    for (int o = W / 4; o > 0; o >>= 1) mine += __shfl_xor_sync(mask, mine, o);
    if constexpr (L == 0) {
      const int warps = blockDim.x >> 5, l = threadIdx.x & 31;
      if (warps > 1) {
        if ((threadIdx.x & 15) == 0) buf[(l >> 4) * 16 + (threadIdx.x >> 5)] = mine;
        __syncthreads();
        mine = (l & 15) < warps ? buf[l] : 0.0f;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1)
          if (o < warps) mine += __shfl_xor_sync(mask, mine, o);
      }
    }
    return make_float2(__shfl_sync(mask, mine, 0, W), __shfl_sync(mask, mine, W / 2, W));
  }
};

// ---- launches -----------------------------------------------------------------------------------
constexpr int kSMs = 148;

// Lets a kernel have `smem` bytes of dynamic shared memory (and its static ones: 48 KB together need no leave) on the current
// device; `done`: a bit per device that was seen.
template <class K>
void allow_smem(K kernel, int smem, std::atomic<uint64_t>& done) {
  int device = 0;
  if (smem <= 46 << 10 || cudaGetDevice(&device) != cudaSuccess) return;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (done.load(std::memory_order_relaxed) & bit) return;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
}

template <class K>
int blocks_per_sm(K kernel, int threads, int smem) {
  int n = 0;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) == cudaSuccess && n > 0 ? n : 1;
}

inline int clamp_blocks(int64_t wanted, int64_t most) { return (int)std::max<int64_t>(1, std::min(wanted, most)); }

}  // namespace
}  // namespace rof
