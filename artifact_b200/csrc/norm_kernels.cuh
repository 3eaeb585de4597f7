// Device code of norm.cu, one translation unit per element type (norm_f32.cu, norm_bf16.cu, norm_f16.cu).
//
// All of it moves a few bytes per operation and is bound by HBM, so the layout is about keeping 16-byte loads in
// flight.  A *group* of L threads owns one row at a time and lane i of it the vectors i, i + L, ... of the row (L = 4..32
// inside a warp, or the whole block for wide rows); weights, biases and the column sums of the backward
// pass stay in the thread's registers over all its rows.
//
// Rows that do not start on a 16-byte boundary use the same vectors: vector i of a row starts at column i * VEC - s, where s is
// the row start's distance from the boundary below it; the first and last vector then hold some of their neighbours' elements,
// which are cleared after the load and not written.  s has period VEC in the row number, and the groups advance by a multiple of
// VEC rows, so a thread's columns never change.  The inputs of a call must share s; an output that lies differently is
// written through shared memory.  What is left — inputs that lie differently, rows of more than 8,192 columns — runs on the
// *_plain kernels.  (Contiguous matrices of up to 511 columns whose rows are not whole vectors: norm_tile.cuh.)
//
// Measured on B200, of the measured copy bandwidth (6,460 GB/s; every matrix read or written once per pass): layer norm
// 2449029x256 fp32 forward 764 us (102 %), back 1,180 us (99 %); 232965x602 fp32 178 us (98 %), 287 us (91 %); 16384x4096
// bf16 52 us (80 %), 89 us (70 %: a block per row and few warps to cover its two sums).  With the ReLU and the generator in 16 bits neither
// DRAM nor the issue slots are full (1000000x64 bf16: 74 us, 53 %; 103 us, 58 %): two blocks of 256 threads an SM do not cover the
// row's chain of sums and rounds.  Padded rows beside contiguous ones: 200000x301 fp32 80 and 130 us (93 and 86 %), 1000000x47
// bf16 100 and 105 us (29 and 41 %).  The *_plain kernels: 30000x10000 fp32 1,056 and 2,107 us (35 and 26 %).
#pragma once
#include "norm_device.cuh"

namespace rof {
namespace {

// distance of row r's first element from the 16-byte boundary below it
template <class T, bool EDGE>
__device__ __forceinline__ int row_shift(const void* base, int64_t ld, int64_t r) {
  if constexpr (!EDGE) return 0;
  return (int)((reinterpret_cast<uintptr_t>(base) / sizeof(T) + (uint64_t)(r * ld)) % kVec<T>);
}

// How the rows of the matrices lie: whole 16-byte vectors; with partial vectors at the ends, the same in all of them; or the inputs
// alike and the output differently.
enum { kWhole, kEdges, kMoved };

// Threads of a block that owns a row: at most this many, so that 16 elements a thread have 128 registers and 32 have 255.
template <class T, int C>
constexpr int wide_threads() { return C * kVec<T> <= 16 ? 512 : 256; }

// The forward pass runs two blocks of 256 threads per SM and no more: with the rings, 512 threads keep enough in flight, and more of
// them only mix their reads and writes more finely (2449029x256 fp32: 760 us with two, 834 with three, 956 with one).
constexpr int kForwardBlocks = 2;
// Blocks of 256 threads per SM that the register allocation aims at.  Backward: as many as spill at most 8 bytes (rows of a block have
// registers of their own, wide_threads(), and up to 92).  Forward: two; one for 32 elements a thread with the generator and partial vectors,
// which would spill 400 bytes with two (200000x1001 fp32: 351 us, 433 with two).  At 24 elements two blocks spill 120 bytes and are
// faster all the same (300000x601 bf16 331 us, 394 with one; with padded rows, 200 bytes, 436 and 488, but 500000x300 314 and 296); at 20
// they spill 8 (60 with padded rows; 300000x602 fp32 261 and 352).
template <class T, int C, bool HIDDEN, bool EDGE>
constexpr int forward_blocks() { return HIDDEN && EDGE && C * kVec<T> > 24 ? 1 : kForwardBlocks; }
template <class T, int C, bool HIDDEN>
constexpr int backward_blocks() { return C * kVec<T> <= 8 ? (HIDDEN ? 2 : 3) : C * kVec<T> <= (HIDDEN ? 8 : 16) ? 2 : 1; }
// Slots of the rings.  In the forward pass 32-bit rows do best with little in flight (2 slots of 64 bytes a thread and more: 65536x2048 172 us
// against 191 with 3), 16-bit rows, which take more instructions a byte, with more (16384x4096 51 us with 4, 54 with 3).
template <class T, int C, bool BACK>
constexpr int ring_slots() {
  if (BACK) return C == 1 ? 4 : C <= 4 ? 3 : 2;
  if (sizeof(T) == 2) return C == 3 ? 3 : 4;
  return C == 1 ? 4 : C == 2 ? 3 : 2;
}

// ---- layer norm ---------------------------------------------------------------------------------
// the thread's entries of a vector (`other` where there is none)
template <class T, int C>
__device__ __forceinline__ void load_columns(float2 (&out)[C][kVec<T> / 2], const void* p, int f32, int dim, int c0, int advance, float other) {
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int t = 0; t < kVec<T> / 2; ++t) {
      const int c = c0 + k * advance + 2 * t;
      out[k][t].x = p != nullptr && (unsigned)c < (unsigned)dim ? vector_at<T>(p, f32, c) : other;
      out[k][t].y = p != nullptr && (unsigned)(c + 1) < (unsigned)dim ? vector_at<T>(p, f32, c + 1) : other;
    }
}

// how many rows first, first + stride, ... there are
__device__ __forceinline__ int rows_of(int64_t rows, int64_t first, int64_t stride) {
  return first < rows ? (int)((rows - first + stride - 1) / stride) : 0;
}

// What is computed from v is computed where it is used: the comparisons of a thread's columns with the ends of the row do not
// change from row to row, but kept over the loop they cost more registers than the row itself.
__device__ __forceinline__ void not_hoisted(int& v) { asm volatile("" : "+r"(v)); }

// HIDDEN: with the ReLU or the dropout (or both)
template <class T, int L, int C, bool HIDDEN, int LAYOUT>
__global__ void __launch_bounds__(L == 0 ? wide_threads<T, C>() : 256, L == 0 ? 1 : forward_blocks<T, C, HIDDEN, LAYOUT != kWhole>()) norm_forward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int V = kVec<T>, H = V / 2;
  constexpr bool EDGE = LAYOUT != kWhole;
  __shared__ float buf[2][32];
  extern __shared__ uint4 ring_memory[];
  const Group<L> g;
  const int s = row_shift<T, EDGE>(a.x, a.ldx, g.first);
  int c0 = g.lane * V - s;
  const int advance = g.lanes * V;
  const uint64_t step = HIDDEN ? step_of(a.drop) : 0;
  const float inv = 1.0f / (float)a.dim;
  constexpr int S = ring_slots<T, C, false>();
  const int rows = rows_of(a.rows, g.first, g.stride);
  Ring<T, L, C, S, EDGE> ring(ring_memory, 0, a.x, a.ldx, g.first, g.stride, c0, g.lanes, a.dim);
  const int slot_bytes = ring.slot_bytes();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < rows) ring.fetch(i * slot_bytes);
    copy_commit();
  }
  float2 w[C][H], b[C][H];
  load_columns<T, C>(w, a.weight, a.wf32, a.dim, c0, advance, 1.0f);
  load_columns<T, C>(b, a.bias, a.wf32, a.dim, c0, advance, 0.0f);
  const bool ragged = EDGE || a.dim != g.lanes * C * V;            // some threads hold less than C vectors of the row
  int at = 0, next = (S - 1) * slot_bytes;         // the slot to read and the one to fill
  T* y = reinterpret_cast<T*>(a.out) + g.first * a.ldo;
  // two elements at a time where both sides allow it
  const bool pairs = LAYOUT == kMoved && a.dim % 2 == 0 && s % 2 == 0 && a.ldo % 2 == 0 && reinterpret_cast<uintptr_t>(a.out) % (2 * sizeof(T)) == 0;
  const int64_t y_step = g.stride * a.ldo, e_step = g.stride * a.dim;
  float2* stats = a.stats != nullptr ? a.stats + g.first : nullptr;
  int64_t e = HIDDEN ? a.drop.first + g.first * a.dim + c0 : 0;
  for (int i = 0; i < rows; ++i) {
    if constexpr (EDGE) not_hoisted(c0);
    Pack<T> raw[C];
    copy_wait<S - 2>();
    ring.read(at, raw, c0);
    if (i + S - 1 < rows) ring.fetch(next);
    copy_commit();
    next = at;
    at = at == (S - 1) * slot_bytes ? 0 : at + slot_bytes;
    float2 v[C][H], total = both(0.0f);
#pragma unroll
    for (int k = 0; k < C; ++k) {
      unpack<T>(raw[k], v[k]);
#pragma unroll
      for (int t = 0; t < H; ++t) total = __fadd2_rn(total, v[k][t]);
    }
    // the mean, corrected by the sum of the deviations from its first value
    float mean = g.sum(total.x + total.y, buf[0]) * inv;
    float2 dev1 = both(0.0f), dev2 = both(0.0f), minus = both(-mean);
    if (ragged) {                                   // what lies outside the row deviates by nothing
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const int c = c0 + k * advance;
        if (!EDGE) {
#pragma unroll
          for (int t = 0; t < H; ++t) v[k][t] = c < a.dim ? v[k][t] : both(mean);
        } else if (c < 0 || c + V > a.dim) {
#pragma unroll
          for (int t = 0; t < H; ++t) {
            if ((unsigned)(c + 2 * t) >= (unsigned)a.dim) v[k][t].x = mean;
            if ((unsigned)(c + 2 * t + 1) >= (unsigned)a.dim) v[k][t].y = mean;
          }
        }
      }
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
#pragma unroll
      for (int t = 0; t < H; ++t) {
        const float2 d = __fadd2_rn(v[k][t], minus);
        dev1 = __fadd2_rn(dev1, d);
        dev2 = __ffma2_rn(d, d, dev2);
      }
    }
    const float2 dev = g.sum(make_float2(dev1.x + dev1.y, dev2.x + dev2.y), buf[1]);
    const float off = dev.x * inv;
    mean += off;
    minus = both(-mean);
    const float rstd = rsqrt_of(variance_of(dev.y * inv, off) + a.eps);
    if (stats != nullptr) {
      if (g.lane == 0) *stats = make_float2(mean, rstd);
      stats += g.stride;
    }
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int t = 0; t < H; ++t) v[k][t] = __ffma2_rn(__fmul2_rn(__fadd2_rn(v[k][t], minus), both(rstd)), w[k][t], b[k][t]);
    if constexpr (HIDDEN) {
      if (a.relu) {
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int t = 0; t < H; ++t) v[k][t] = make_float2(relu_of(v[k][t].x), relu_of(v[k][t].y));
      }
      if (a.drop.on) {
        uint32_t words[C * V];
        draw_words<C, V, EDGE>(a.drop, step, e, advance, words);
        e += e_step;
        scale_elements(v, a.drop.scale);
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int t = 0; t < H; ++t) v[k][t] = kept_of(a.drop, words + k * V + 2 * t, v[k][t]);
      }
    }
    if constexpr (LAYOUT == kMoved) {
      if (pairs) ring.template store_through<2>(next, v, g, y, s, a.dim);
      else ring.template store_through<1>(next, v, g, y, s, a.dim);
    } else {
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (c0 + k * advance < a.dim) store_vec<T, EDGE>(y, c0 + k * advance, a.dim, v[k]);
    }
    y += y_step;
  }
}

// Sums the groups' column sums of a block in order and stores them: out[c] for c in [0, dim).  Group i holds its
// vectors' elements in `acc`; its columns are shifted by shift(i).
template <class T, int L, int C, bool EDGE>
__device__ __forceinline__ void store_columns(const float2 (&acc)[C][kVec<T> / 2], const Group<L>& g, float* out, int dim,
                                              const void* base, int64_t ld, float* smem) {
  constexpr int V = kVec<T>;
  if constexpr (L == 0) {
    const int s = row_shift<T, EDGE>(base, ld, g.first);
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int t = 0; t < V; ++t) {
        const int c = (g.lane + k * g.lanes) * V - s + t;
        if ((unsigned)c < (unsigned)dim) out[c] = half_of(acc[k][t / 2], t % 2);
      }
  } else {
    constexpr int kWidth = L * C * V, kGroups = 256 / L;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int t = 0; t < V; ++t) smem[g.index * kWidth + (g.lane + k * L) * V + t] = half_of(acc[k][t / 2], t % 2);
    __syncthreads();
    for (int c = threadIdx.x; c < dim; c += 256) {
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < kGroups; ++i)
        sum += smem[i * kWidth + c + row_shift<T, EDGE>(base, ld, (int64_t)blockIdx.x * kGroups + i)];
      out[c] = sum;
    }
  }
}

// dx of every row, and per block the sums over its rows of dz h and dz: partial[block][2][dim]
template <class T, int L, int C, bool HIDDEN, int LAYOUT>
__global__ void __launch_bounds__(L == 0 ? wide_threads<T, C>() : 256, L == 0 ? 1 : backward_blocks<T, C, HIDDEN>()) norm_backward_kernel(const __grid_constant__ NormArgs a) {
  constexpr int V = kVec<T>, H = V / 2;
  constexpr bool EDGE = LAYOUT != kWhole;
  __shared__ float buf[2][32];
  extern __shared__ uint4 ring_memory[];
  const Group<L> g;
  const int s = row_shift<T, EDGE>(a.x, a.ldx, g.first);
  int c0 = g.lane * V - s;
  const int advance = g.lanes * V;
  const uint64_t step = HIDDEN ? step_of(a.drop) : 0;
  const float inv = 1.0f / (float)a.dim;
  constexpr int S = ring_slots<T, C, true>();
  const int rows = rows_of(a.rows, g.first, g.stride);
  Ring<T, L, C, S, EDGE> ring_x(ring_memory, 0, a.x, a.ldx, g.first, g.stride, c0, g.lanes, a.dim);
  Ring<T, L, C, S, EDGE> ring_dy(ring_memory, 1, a.dy, a.lddy, g.first, g.stride, c0, g.lanes, a.dim);
  const int slot_bytes = ring_x.slot_bytes();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < rows) {
      ring_x.fetch(i * slot_bytes);
      ring_dy.fetch(i * slot_bytes);
    }
    copy_commit();
  }
  const float2* stats = a.stats + g.first;
  float2 st_next = rows > 0 ? *stats : both(0.0f);
  float2 w[C][H], b[HIDDEN ? C : 1][H], aw[C][H], ab[C][H];
  load_columns<T, C>(w, a.weight, a.wf32, a.dim, c0, advance, 1.0f);
  if constexpr (HIDDEN) load_columns<T, C>(b, a.relu ? a.bias : nullptr, a.wf32, a.dim, c0, advance, 0.0f);
#pragma unroll
  for (int k = 0; k < C; ++k)
#pragma unroll
    for (int t = 0; t < H; ++t) aw[k][t] = ab[k][t] = both(0.0f);
  int turn = 0, at = 0, next = (S - 1) * slot_bytes;
  T* dx = reinterpret_cast<T*>(a.out) + g.first * a.ldo;
  const bool pairs = LAYOUT == kMoved && a.dim % 2 == 0 && s % 2 == 0 && a.ldo % 2 == 0 && reinterpret_cast<uintptr_t>(a.out) % (2 * sizeof(T)) == 0;
  const int64_t dx_step = g.stride * a.ldo, e_step = g.stride * a.dim;
  int64_t e = HIDDEN ? a.drop.first + g.first * a.dim + c0 : 0;
  for (int i = 0; i < rows; ++i, turn ^= 1) {
    if constexpr (EDGE) not_hoisted(c0);
    const float2 st = st_next;
    stats += g.stride;
    if (i + 1 < rows) st_next = *stats;
    uint32_t words[HIDDEN ? C * V : 1];             // drawn while the row is on its way
    if constexpr (HIDDEN) {
      if (a.drop.on) draw_words<C, V, EDGE>(a.drop, step, e, advance, words);
      e += e_step;
    }
    Pack<T> rx[C], rd[C];
    copy_wait<S - 2>();
    ring_x.read(at, rx, c0);
    ring_dy.read(at, rd, c0);
    if (i + S - 1 < rows) {
      ring_x.fetch(next);
      ring_dy.fetch(next);
    }
    copy_commit();
    next = at;
    at = at == (S - 1) * slot_bytes ? 0 : at + slot_bytes;
    const float2 minus = both(-st.x), rstd = both(st.y);
    float2 h[C][H], gr[C][H], s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int k = 0; k < C; ++k) unpack<T>(rd[k], gr[k]);
    if constexpr (HIDDEN) {
      if (a.drop.on) {
        scale_elements(gr, a.drop.scale);
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int t = 0; t < H; ++t) gr[k][t] = kept_of(a.drop, words + k * V + 2 * t, gr[k][t]);
      }
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      unpack<T>(rx[k], h[k]);
#pragma unroll
      for (int t = 0; t < H; ++t) {
        // (a column outside the row has x = dy = 0 and adds nothing anywhere)
        h[k][t] = __fmul2_rn(__fadd2_rn(h[k][t], minus), rstd);
        float2 dz = gr[k][t];
        if constexpr (HIDDEN) {
          if (a.relu) {
            const float2 z = __ffma2_rn(h[k][t], w[k][t], b[k][t]);
            dz = make_float2(z.x <= 0.0f ? 0.0f : dz.x, z.y <= 0.0f ? 0.0f : dz.y);
          }
        }
        aw[k][t] = __ffma2_rn(dz, h[k][t], aw[k][t]);
        ab[k][t] = __fadd2_rn(ab[k][t], dz);
        gr[k][t] = __fmul2_rn(dz, w[k][t]);
        s1 = __fadd2_rn(s1, gr[k][t]);
        s2 = __ffma2_rn(gr[k][t], h[k][t], s2);
      }
    }
    if (a.out == nullptr) continue;
    const float2 sums = g.sum(make_float2(s1.x + s1.y, s2.x + s2.y), buf[turn]);
    const float2 c1 = both(-sums.x * inv), c2 = both(-sums.y * inv);
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int t = 0; t < H; ++t) gr[k][t] = __fmul2_rn(__fadd2_rn(gr[k][t], __ffma2_rn(h[k][t], c2, c1)), rstd);
    if constexpr (LAYOUT == kMoved) {
      if (pairs) ring_x.template store_through<2>(next, gr, g, dx, s, a.dim);
      else ring_x.template store_through<1>(next, gr, g, dx, s, a.dim);
    } else {
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (c0 + k * advance < a.dim) store_vec<T, EDGE>(dx, c0 + k * advance, a.dim, gr[k]);
    }
    dx += dx_step;
  }
  if (a.partial != nullptr) {
    copy_wait<0>();                                 // the groups' sums go where the ring was
    float* columns = reinterpret_cast<float*>(ring_memory);
    float* p = a.partial + (int64_t)blockIdx.x * 2 * a.dim;
    store_columns<T, L, C, EDGE>(aw, g, p, a.dim, a.x, a.ldx, columns);
    store_columns<T, L, C, EDGE>(ab, g, p + a.dim, a.dim, a.x, a.ldx, columns);
  }
}

// out[i] = sum over the blocks' partial[block][i] for i in [0, width): eight runs of blocks per column, added in order.  Columns
// up to `split` go to `first`, the others to `second`.
template <class T>
__global__ void __launch_bounds__(256) join_columns_kernel(const float* partial, int blocks, int64_t width, int64_t split, void* first, void* second, int f32) {
  __shared__ float part[8][33];
  const int x = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + x;
  float sum = 0.0f;
  partial += i;
  if (i < width) {
#pragma unroll 8
    for (int k = run; k < blocks; k += 8) sum += partial[k * width];
  }
  part[run][x] = sum;
  __syncthreads();
  if (run == 0 && i < width) {
#pragma unroll
    for (int k = 1; k < 8; ++k) sum += part[k][x];
    void* out = i < split ? first : second;
    if (out != nullptr) vector_put<T>(out, f32, (int)(i < split ? i : i - split), sum);
  }
}

// ---- layer norm, any alignment and width ---------------------------------------------------------
// One block per row and one element per load, for matrices whose rows lie differently against the 16-byte boundaries and for rows
// wider than a block's registers; the row is read again instead of kept.
template <class T>
__global__ void __launch_bounds__(256) norm_forward_plain(const __grid_constant__ NormArgs a) {
  __shared__ float buf[2][32];
  const Group<0> g;
  const uint64_t step = step_of(a.drop);
  const float inv = 1.0f / (float)a.dim;
  for (int64_t r = g.first; r < a.rows; r += g.stride) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    T* y = reinterpret_cast<T*>(a.out) + r * a.ldo;
    float total = 0.0f;
    for (int c = g.lane; c < a.dim; c += g.lanes) total += to_float(x[c]);
    float mean = g.sum(total, buf[0]) * inv;
    float2 dev = make_float2(0.0f, 0.0f);
    for (int c = g.lane; c < a.dim; c += g.lanes) {
      const float d = to_float(x[c]) - mean;
      dev.x += d;
      dev.y = __fmaf_rn(d, d, dev.y);
    }
    dev = g.sum(dev, buf[1]);
    const float off = dev.x * inv;
    mean += off;
    const float rstd = rsqrt_of(variance_of(dev.y * inv, off) + a.eps);
    if (a.stats != nullptr && g.lane == 0) a.stats[r] = make_float2(mean, rstd);
    for (int c = g.lane; c < a.dim; c += g.lanes) {
      float z = affine((to_float(x[c]) - mean) * rstd, a.weight != nullptr ? vector_at<T>(a.weight, a.wf32, c) : 1.0f,
                       a.bias != nullptr ? vector_at<T>(a.bias, a.wf32, c) : 0.0f);
      if (a.relu) z = relu_of(z);
      if (a.drop.on) z = kept(a.drop, step, a.drop.first + r * a.dim + c) ? z * a.drop.scale : 0.0f;
      y[c] = from_float<T>(z);
    }
  }
}

template <class T>
__device__ __forceinline__ float norm_dz(const NormArgs& a, uint64_t step, int64_t r, int c, float h, float w) {
  float dz = to_float(reinterpret_cast<const T*>(a.dy)[r * a.lddy + c]);
  if (a.drop.on) dz = kept(a.drop, step, a.drop.first + r * a.dim + c) ? dz * a.drop.scale : 0.0f;
  if (a.relu && affine(h, w, a.bias != nullptr ? vector_at<T>(a.bias, a.wf32, c) : 0.0f) <= 0.0f) dz = 0.0f;
  return dz;
}

template <class T>
__global__ void __launch_bounds__(256) norm_backward_rows_plain(const __grid_constant__ NormArgs a) {
  __shared__ float buf[2][32];
  const Group<0> g;
  const uint64_t step = step_of(a.drop);
  const float inv = 1.0f / (float)a.dim;
  int turn = 0;
  for (int64_t r = g.first; r < a.rows; r += g.stride, turn ^= 1) {
    const T* x = reinterpret_cast<const T*>(a.x) + r * a.ldx;
    T* dx = reinterpret_cast<T*>(a.out) + r * a.ldo;
    const float2 st = a.stats[r];
    float2 sums = make_float2(0.0f, 0.0f);
    for (int c = g.lane; c < a.dim; c += g.lanes) {
      const float h = (to_float(x[c]) - st.x) * st.y, w = a.weight != nullptr ? vector_at<T>(a.weight, a.wf32, c) : 1.0f;
      const float gr = w * norm_dz<T>(a, step, r, c, h, w);
      sums.x += gr;
      sums.y = __fmaf_rn(gr, h, sums.y);
    }
    sums = g.sum(sums, buf[turn]);
    const float c1 = sums.x * inv, c2 = sums.y * inv;
    for (int c = g.lane; c < a.dim; c += g.lanes) {
      const float h = (to_float(x[c]) - st.x) * st.y, w = a.weight != nullptr ? vector_at<T>(a.weight, a.wf32, c) : 1.0f;
      dx[c] = from_float<T>(st.y * (w * norm_dz<T>(a, step, r, c, h, w) - __fmaf_rn(h, c2, c1)));
    }
  }
}

// thread = column, blockIdx.y = a run of rows
template <class T>
__global__ void __launch_bounds__(128) norm_backward_columns_plain(const __grid_constant__ NormArgs a, int64_t run_rows) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= a.dim) return;
  const uint64_t step = step_of(a.drop);
  const float w = a.weight != nullptr ? vector_at<T>(a.weight, a.wf32, c) : 1.0f;
  const int64_t r0 = (int64_t)blockIdx.y * run_rows, r1 = min(a.rows, r0 + run_rows);
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const float2 st = a.stats[r];
    const float h = (to_float(reinterpret_cast<const T*>(a.x)[r * a.ldx + c]) - st.x) * st.y;
    const float dz = norm_dz<T>(a, step, r, c, h, w);
    s1 = __fmaf_rn(dz, h, s1);
    s2 += dz;
  }
  a.partial[((int64_t)blockIdx.y * 2 + 0) * a.dim + c] = s1;
  a.partial[((int64_t)blockIdx.y * 2 + 1) * a.dim + c] = s2;
}

// ---- dropout ------------------------------------------------------------------------------------
// U vectors that lie `advance` elements apart, e the index of the first.  BACK = false: drop(relu?(x + b)); BACK = true: dy behind the
// dropout and the ReLU, where with the ReLU the forward's output y says which elements were kept and positive.  DRAW: the
// generator is asked.
template <class T, int U, bool BACK, bool DRAW, bool BIAS, bool EDGE>
__device__ __forceinline__ void drop_vectors(const DropArgs& a, uint64_t step, int64_t e, int64_t advance, const Pack<T> (&in)[U],
                                             const Pack<T> (&y)[U], const float2 (&b)[kVec<T> / 2], float2 (&o)[U][kVec<T> / 2]) {
  constexpr int V = kVec<T>, H = V / 2;
  constexpr bool MARK = !BACK && BIAS && sizeof(T) == 2;       // the ReLU follows at the store
#pragma unroll
  for (int u = 0; u < U; ++u) {
    unpack<T>(in[u], o[u]);
    if constexpr (BACK) {
      if (!DRAW && a.relu) {
        float2 f[H];
        unpack<T>(y[u], f);
#pragma unroll
        for (int t = 0; t < H; ++t) o[u][t] = make_float2(passed_of(f[t].x, o[u][t].x), passed_of(f[t].y, o[u][t].y));
      }
    } else {
      if constexpr (BIAS) {
#pragma unroll
        for (int t = 0; t < H; ++t) o[u][t] = __fadd2_rn(o[u][t], b[t]);
      }
      if (!MARK && a.relu) {
#pragma unroll
        for (int t = 0; t < H; ++t) o[u][t] = make_float2(relu_of(o[u][t].x), relu_of(o[u][t].y));
      }
    }
  }
  if constexpr (MARK) scaled<T>(o, a.drop.scale, a.relu);
  else scale_elements(o, a.drop.scale);
  if constexpr (DRAW) {
    const float dropped = MARK && a.relu ? -0.0f : 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t words[V];
      draw_words<1, V, EDGE>(a.drop, step, e + u * advance, 0, words);
#pragma unroll
      for (int t = 0; t < H; ++t) o[u][t] = kept_of(a.drop, words + 2 * t, o[u][t], dropped);
    }
  }
}

// Contiguous matrices without a bias: one run of n elements from an aligned address.  A block takes U x 256 vectors side by side and
// is done: U = 4 vectors a thread (2 where two matrices are read) are enough calls to fill the generator's chains.  Bound by HBM in 32 bits;
// in 16, with the generator, the issue slots are 58-62 % busy beside 59-63 % of DRAM.
template <class T, bool BACK, bool DRAW, bool EDGE>
__global__ void __launch_bounds__(256, 4) dropout_flat_kernel(const __grid_constant__ DropArgs a, int64_t n) {
  constexpr int V = kVec<T>, U = BACK && !DRAW ? 2 : 4;
  const uint64_t step = DRAW ? step_of(a.drop) : 0;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* y = reinterpret_cast<const T*>(a.y);
  T* out = reinterpret_cast<T*>(a.out);
  const bool two = BACK && !DRAW && a.relu;
  const float2 zero[V / 2] = {};
  const int64_t vectors = n / V, i = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
  Pack<T> in[U], yy[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    in[u].raw = yy[u].raw = make_uint4(0, 0, 0, 0);
    if (i + u * 256 < vectors) {
      in[u].raw = reinterpret_cast<const uint4*>(x)[i + u * 256];
      if (two) yy[u].raw = reinterpret_cast<const uint4*>(y)[i + u * 256];
    }
  }
  float2 o[U][V / 2];
  drop_vectors<T, U, BACK, DRAW, false, EDGE>(a, step, a.drop.first + i * V, 256 * V, in, yy, zero, o);
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (i + u * 256 < vectors) store_vec<T, false>(out + (i + u * 256) * V, 0, V, o[u]);
  // the last elements that fill no vector
  const int64_t e = vectors * V + threadIdx.x;
  if (blockIdx.x == 0 && e < n) {
    float z = to_float(x[e]);
    const bool keep = !DRAW || kept(a.drop, step, a.drop.first + e);
    if (!BACK && a.relu) z = relu_of(z);
    if (two && !passed(y[e])) z = 0.0f;
    out[e] = from_float<T>(keep ? z * a.drop.scale : 0.0f);
  }
}

// Rows that a thread of dropout_rows_kernel takes at once, and blocks per SM that its registers aim at.  With the generator, sixteen
// elements; behind a ReLU the backward pass only streams, and whole 32-bit vectors do it with many warps (232965x256:
// 124 us, 133 with four rows and four blocks), 16-bit ones with many rows (1000000x64 bf16: 73 us, 86).
template <class T, bool STREAM, bool EDGE>
constexpr int drop_rows_at_once() { return !STREAM ? 16 / kVec<T> : sizeof(T) == 2 ? 8 : EDGE ? 4 : 2; }
template <class T, bool STREAM, bool EDGE>
constexpr int drop_row_blocks() { return !STREAM ? 3 : sizeof(T) == 2 ? 2 : EDGE ? 3 : 6; }

// Thread = vector `c` of the rows first, first + stride, ...; a.lanes threads side by side cover a tile of a row.  U rows at a time:
// their loads and their calls of the generator run side by side.
template <class T, bool BACK, bool DRAW, bool EDGE>
__global__ void __launch_bounds__(256, drop_row_blocks<T, BACK && !DRAW, EDGE>()) dropout_rows_kernel(const __grid_constant__ DropArgs a) {
  constexpr int V = kVec<T>, U = drop_rows_at_once<T, BACK && !DRAW, EDGE>();
  extern __shared__ float columns[];
  const int groups = blockDim.x / a.lanes, group = threadIdx.x / a.lanes, lane = threadIdx.x - group * a.lanes;
  const int64_t first = (int64_t)blockIdx.x * groups + group, stride = (int64_t)gridDim.x * groups;
  const int s = row_shift<T, EDGE>(a.x, a.ldx, first);
  const int c = (int)(blockIdx.y * a.lanes + lane) * V - s;
  const bool live = group < groups && c < a.dim;
  const uint64_t step = DRAW ? step_of(a.drop) : 0;
  const bool two = BACK && !DRAW && a.relu;
  float2 b[1][V / 2], acc[V / 2];
  load_columns<T, 1>(b, !BACK && live ? a.bias : nullptr, a.bf32, a.dim, c, 0, 0.0f);
#pragma unroll
  for (int t = 0; t < V / 2; ++t) acc[t] = both(0.0f);
  if (live) {
    for (int64_t r = first; r < a.rows; r += U * stride) {
      Pack<T> in[U], yy[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        in[u].raw = yy[u].raw = make_uint4(0, 0, 0, 0);
        if (r + u * stride < a.rows) {
          load_vec<T, EDGE>(in[u], reinterpret_cast<const T*>(a.x) + (r + u * stride) * a.ldx, c, a.dim, r + u * stride, a.rows);
          if (two) load_vec<T, EDGE>(yy[u], reinterpret_cast<const T*>(a.y) + (r + u * stride) * a.ldy, c, a.dim, r + u * stride, a.rows);
        }
      }
      float2 o[U][V / 2];
      drop_vectors<T, U, BACK, DRAW, true, EDGE>(a, step, a.drop.first + r * a.dim + c, stride * a.dim, in, yy, b[0], o);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (r + u * stride < a.rows) {
          if constexpr (BACK) {
#pragma unroll
            for (int t = 0; t < V / 2; ++t) acc[t] = __fadd2_rn(acc[t], o[u][t]);
          }
          if (a.out != nullptr) store_vec<T, EDGE>(reinterpret_cast<T*>(a.out) + (r + u * stride) * a.ldo, c, a.dim, o[u], !BACK && a.relu);
        }
    }
  }
  if (!BACK || a.partial == nullptr) return;
  if (group < groups) {
#pragma unroll
    for (int t = 0; t < V; ++t) columns[(group * a.lanes + lane) * V + t] = live ? half_of(acc[t / 2], t % 2) : 0.0f;
  }
  __syncthreads();
  const int tile = a.lanes * V, c0 = blockIdx.y * tile;
  // Group k holds columns [c0 - shift, c0 - shift + tile).  With more than one tile a block has one group, so the tiles' columns
  // neither overlap nor leave a gap.
  float* p = a.partial + (int64_t)blockIdx.x * a.dim;
  for (int i = threadIdx.x; i < tile + (EDGE ? V : 0); i += blockDim.x) {
    float sum = 0.0f;
    const int col = c0 - (EDGE ? V : 0) + i;
    bool any = false;
    for (int k = 0; k < groups; ++k) {
      const int j = col - c0 + row_shift<T, EDGE>(a.x, a.ldx, (int64_t)blockIdx.x * groups + k);
      if (j >= 0 && j < tile) {
        sum += columns[k * tile + j];
        any = true;
      }
    }
    if (any && (unsigned)col < (unsigned)a.dim) p[col] = sum;
  }
}

// Any layout: a thread takes the four elements of a call of the generator (fewer at the matrix's ends), U times; they may lie in two
// rows or more.  `whole`: bit 0: x, bit 1: y, bit 2: out are contiguous and their groups of four aligned to their size.
template <class T, bool BACK>
__global__ void __launch_bounds__(256, 4) dropout_any_kernel(const __grid_constant__ DropArgs a, int whole) {
  constexpr int U = 2;
  const uint64_t step = step_of(a.drop);
  constexpr bool MARK = !BACK && sizeof(T) == 2;
  const bool two = BACK && a.relu, draw = a.drop.on && !two, mark = MARK && a.relu;
  const int64_t n = a.rows * a.dim, ahead = a.drop.first & 3;         // element 0 is number `ahead` of its group
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t i0 = (((int64_t)blockIdx.x * U + u) * 256 + threadIdx.x) * 4 - ahead;
    if (i0 >= n) return;
    const int from = i0 < 0 ? (int)-i0 : 0, to = (int)min((int64_t)4, n - i0);
    int64_t r = (i0 + from) / a.dim;
    int c = (int)(i0 + from - r * a.dim);
    const bool full = from == 0 && to == 4;
    uint4 w = make_uint4(0, 0, 0, 0);
    if (draw) w = philox7((uint64_t)(a.drop.first + i0) >> 2, step, a.drop.key);
    const uint32_t words[4] = {w.x, w.y, w.z, w.w};
    alignas(16) T in[4];
    alignas(16) T y[4];
    alignas(16) T out[4];
    if (full && (whole & 1)) four_copy(in, reinterpret_cast<const T*>(a.x) + i0);
    if (full && two && (whole & 2)) four_copy(y, reinterpret_cast<const T*>(a.y) + i0);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      if (t < from || t >= to) continue;
      if (!(full && (whole & 1))) in[t] = reinterpret_cast<const T*>(a.x)[r * a.ldx + c];
      if (two && !(full && (whole & 2))) y[t] = reinterpret_cast<const T*>(a.y)[r * a.ldy + c];
      float z = to_float(in[t]);
      if constexpr (BACK) {
        if (two && !passed(y[t])) z = 0.0f;
        z *= a.drop.scale;
      } else {
        if (a.bias != nullptr) z += vector_at<T>(a.bias, a.bf32, c);
        if (!MARK && a.relu) z = relu_of(z);
        z = __fmaf_rn(z, a.drop.scale, mark ? -kLeast : -0.0f);
      }
      out[t] = from_float<T>(draw && words[t] <= a.drop.last ? (mark ? -0.0f : 0.0f) : z);
      if (!(full && (whole & 4))) {
        if constexpr (MARK) {
          if (mark) out[t] = relu_marked_one(out[t]);
        }
        reinterpret_cast<T*>(a.out)[r * a.ldo + c] = out[t];
      }
      if (++c == a.dim) {
        c = 0;
        ++r;
      }
    }
    if constexpr (MARK) {
      if (mark && full && (whole & 4)) {
        uint32_t* pair = reinterpret_cast<uint32_t*>(out);
        pair[0] = relu_marked<T>(pair[0]);
        pair[1] = relu_marked<T>(pair[1]);
      }
    }
    if (full && (whole & 4)) four_copy(reinterpret_cast<T*>(a.out) + i0, out);
  }
}

template <class T>
__global__ void __launch_bounds__(128) dropout_columns_plain(const __grid_constant__ DropArgs a, int64_t run_rows) {
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= a.dim) return;
  const uint64_t step = step_of(a.drop);
  const int64_t r0 = (int64_t)blockIdx.y * run_rows, r1 = min(a.rows, r0 + run_rows);
  float sum = 0.0f;
  for (int64_t r = r0; r < r1; ++r) {
    const bool keep = a.relu ? passed(reinterpret_cast<const T*>(a.y)[r * a.ldy + c])
                             : !a.drop.on || kept(a.drop, step, a.drop.first + r * a.dim + c);
    if (keep) sum += to_float(reinterpret_cast<const T*>(a.x)[r * a.ldx + c]) * a.drop.scale;
  }
  a.partial[(int64_t)blockIdx.y * a.dim + c] = sum;
}

// ---- launches -----------------------------------------------------------------------------------
// How the rows of a call's matrices lie against the 16-byte boundaries.  vec: the same way in all of them; edge: there are
// partial vectors; vectors: of a row, at most.
struct Layout {
  bool vec, edge;
  int vectors;
};

struct Matrix {
  const void* p;
  int64_t ld;
};

template <class T>
Layout layout_of(int64_t rows, int dim, std::initializer_list<Matrix> all) {
  constexpr int V = kVec<T>;
  int start = -1, advance = -1;
  for (const Matrix& m : all) {
    if (m.p == nullptr) continue;
    const int s = (int)(reinterpret_cast<uintptr_t>(m.p) / sizeof(T) % V), d = rows > 1 ? (int)(m.ld % V) : 0;
    if (start >= 0 && (s != start || d != advance)) return {false, true, 0};
    start = s;
    advance = d;
  }
  if (start < 0) start = advance = 0;             // no rows
  int gcd = V;                                    // the rows' starts are congruent modulo this
  while (advance % gcd) gcd /= 2;
  const int most = V - gcd + start % gcd;
  const int shift = advance == 0 ? start : most;
  return {true, dim % V != 0 || shift != 0, (int)(((int64_t)dim + shift + V - 1) / V)};
}

// a block per row
template <class T, int C, class F>
bool wide_rows(int vectors, F&& f) {
  const int threads = ((vectors + C - 1) / C + 31) / 32 * 32;
  if (threads > wide_threads<T, C>()) return false;
  f.template operator()<0, C>(threads);
  return true;
}

// Group width L and vectors per lane C for rows of `vectors` vectors -> f.template operator()<L, C>(block threads).  The
// fewest lanes whose registers hold the row: they have the most bytes in flight each and the fewest steps in the row's sums.  How much a
// lane holds: in 32 bits up to 5 vectors (20 elements: weights, biases and sums beside them leave two blocks an SM), a full warp up to 8 in
// the forward pass, where the next choice is a block per row; in 16 bits up to 3 (24 elements), a full warp up to 4 in the backward pass
// (65536x1024 bf16: 73 us, 87 with a block per row).  Back through a ReLU or a dropout, with biases and words as well, up to 3 vectors in 32
// bits and one in 16, a full warp 5 and 2.  Wider rows have a block each, and a thread of it what wide_threads() has registers for (16-bit
// rows of 97 to 256 vectors forward: 16 elements; 32 would leave a block one or two warps).  So a block owns a row above 1,024
// columns (fp32 forward, 16-bit backward), 768 (16-bit forward), 640 (fp32 backward, with a ReLU or a dropout too) and 512 (16-bit
// backward with one).
enum Pass { kForward, kBackward, kBackwardHidden };
template <class T, Pass PASS, class F>
bool by_width(int vectors, F&& f) {
  if constexpr (PASS == kBackwardHidden && sizeof(T) == 4) {
    if (vectors <= 4) f.template operator()<4, 1>(256);
    else if (vectors <= 8) f.template operator()<4, 2>(256);
    else if (vectors <= 16) f.template operator()<8, 2>(256);
    else if (vectors <= 24) f.template operator()<8, 3>(256);
    else if (vectors <= 32) f.template operator()<16, 2>(256);
    else if (vectors <= 48) f.template operator()<16, 3>(256);
    else if (vectors <= 64) f.template operator()<32, 2>(256);
    else if (vectors <= 96) f.template operator()<32, 3>(256);
    else if (vectors <= 128) f.template operator()<32, 4>(256);
    else if (vectors <= 160) f.template operator()<32, 5>(256);          // (300000x602: 368 us, 445 with a block per row)
    else if (vectors <= 1024) return wide_rows<T, 2>(vectors, f);
    else return wide_rows<T, 4>(vectors, f);
  } else if constexpr (PASS == kBackwardHidden) {
    if (vectors <= 4) f.template operator()<4, 1>(256);
    else if (vectors <= 8) f.template operator()<8, 1>(256);
    else if (vectors <= 16) f.template operator()<16, 1>(256);
    else if (vectors <= 32) f.template operator()<32, 1>(256);
    else if (vectors <= 64) f.template operator()<32, 2>(256);
    else if (vectors <= 512) return wide_rows<T, 1>(vectors, f);
    else return wide_rows<T, 2>(vectors, f);
  } else if constexpr (sizeof(T) == 4) {
    if (vectors <= 4) f.template operator()<4, 1>(256);
    else if (vectors <= 8) f.template operator()<4, 2>(256);
    else if (vectors <= 12) f.template operator()<4, 3>(256);
    else if (vectors <= 16) f.template operator()<4, 4>(256);
    else if (vectors <= 20) f.template operator()<4, 5>(256);
    else if (vectors <= 24) f.template operator()<8, 3>(256);
    else if (vectors <= 32) f.template operator()<8, 4>(256);
    else if (vectors <= 40) f.template operator()<8, 5>(256);
    else if (vectors <= 48) f.template operator()<16, 3>(256);
    else if (vectors <= 64) f.template operator()<16, 4>(256);
    else if (vectors <= 80) f.template operator()<16, 5>(256);
    else if (vectors <= 96) f.template operator()<32, 3>(256);
    else if (vectors <= 128) f.template operator()<32, 4>(256);
    else if (vectors <= 160) f.template operator()<32, 5>(256);
    else if (PASS == kForward && vectors <= 256) f.template operator()<32, PASS == kForward ? 8 : 5>(256);
    else return wide_rows<T, 4>(vectors, f);
  } else {
    if (vectors <= 4) f.template operator()<4, 1>(256);
    else if (vectors <= 8) f.template operator()<4, 2>(256);
    else if (vectors <= 12) f.template operator()<4, 3>(256);
    else if (vectors <= 16) f.template operator()<8, 2>(256);
    else if (vectors <= 24) f.template operator()<8, 3>(256);
    else if (vectors <= 32) f.template operator()<16, 2>(256);
    else if (vectors <= 48) f.template operator()<16, 3>(256);
    else if (vectors <= 64) f.template operator()<32, 2>(256);
    else if (vectors <= 96) f.template operator()<32, 3>(256);
    else if (PASS == kBackward && vectors <= 128) f.template operator()<32, PASS == kBackward ? 4 : 3>(256);
    else if (PASS == kForward && vectors <= 256) return wide_rows<T, 2>(vectors, f);
    else return wide_rows<T, 4>(vectors, f);
  }
  return true;
}

template <class T, bool HIDDEN, int LAYOUT>
struct NormForward {
  const NormArgs& a;
  cudaStream_t stream;
  template <int L, int C>
  void operator()(int threads) const {
    auto kernel = norm_forward_kernel<T, L, C, HIDDEN, LAYOUT>;
    constexpr int per_thread = 16 * C * ring_slots<T, C, false>();
    static std::atomic<uint64_t> seen{0};
    allow_smem(kernel, per_thread * (L == 0 ? wide_threads<T, C>() : 256), seen);
    static const int full = blocks_per_sm(kernel, 256, per_thread * 256);
    constexpr int per = L == 0 ? 1 : 256 / std::max(L, 1);
    const int64_t most = (int64_t)kSMs * std::max(1, std::min(full, kForwardBlocks) * 256 / threads);
    int blocks = clamp_blocks((a.rows + per - 1) / per, most);
    if (L == 0) blocks = (blocks + 7) / 8 * 8;
    kernel<<<blocks, threads, per_thread * threads, stream>>>(a);
  }
};

template <class T, bool HIDDEN, int LAYOUT>
struct NormBackward {
  const NormArgs& a;
  cudaStream_t stream;
  int* blocks;
  template <int L, int C>
  void operator()(int threads) const {
    auto kernel = norm_backward_kernel<T, L, C, HIDDEN, LAYOUT>;
    constexpr int per_thread = std::max(32 * C * ring_slots<T, C, true>(), L == 0 ? 0 : C * kVec<T> * 4);
    static std::atomic<uint64_t> seen{0};
    allow_smem(kernel, per_thread * (L == 0 ? wide_threads<T, C>() : 256), seen);
    static const int full = blocks_per_sm(kernel, 256, per_thread * 256);
    constexpr int per = L == 0 ? 1 : 256 / std::max(L, 1);
    const int64_t most = std::min<int64_t>((int64_t)kSMs * (L == 0 ? std::max(1, full * 256 / threads) : full), column_blocks_cap(a.rows, a.dim));
    *blocks = clamp_blocks((a.rows + per - 1) / per, most);
    if (L == 0) *blocks = *blocks < 8 ? 8 : *blocks / 8 * 8;
    kernel<<<*blocks, threads, per_thread * threads, stream>>>(a);
  }
};

// whether the tile kernels take the call: contiguous matrices from 16-byte boundaries, rows that are not whole vectors
template <class T>
bool tiled(int64_t rows, int dim, std::initializer_list<Matrix> all) {
  if (dim > kTileMaxColumns || dim % kVec<T> == 0) return false;
  for (const Matrix& m : all)
    if (m.p != nullptr && ((reinterpret_cast<uintptr_t>(m.p) & 15) != 0 || (rows > 1 && m.ld != dim))) return false;
  return true;
}

inline TileLauncher tile_launcher(float) { return tile_launcher_f32; }
inline TileLauncher tile_launcher(__nv_bfloat16) { return tile_launcher_bf16; }
inline TileLauncher tile_launcher(__half) { return tile_launcher_f16; }

template <class T>
cudaError_t launch_join(const float* partial, int blocks, int64_t width, int64_t split, void* first, void* second, int f32, cudaStream_t stream) {
  join_columns_kernel<T><<<(unsigned)((width + 31) / 32), 256, 0, stream>>>(partial, blocks, width, split, first, second, f32);
  return cudaGetLastError();
}

// (a single row has no row stride; the kernels' shifts of rows that do not exist must not depend on one)
inline NormArgs one_row(NormArgs a) {
  if (a.rows <= 1) a.ldx = a.lddy = a.ldo = 0;
  return a;
}

template <class T>
cudaError_t launch_norm_forward(const NormArgs& given, cudaStream_t stream) {
  const NormArgs a = one_row(given);
  if (tiled<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.out, a.ldo}})) {
    const RowRunArgs t{a.x, nullptr, a.out, a.weight, a.bias, a.wf32, a.stats, nullptr, a.rows, a.dim, a.eps, a.relu, a.drop};
    return tile_launcher(T{})(t, a.relu || a.drop.on ? kNormForwardHidden : kNormForward, stream, nullptr);
  }
  const Layout l = layout_of<T>(a.rows, a.dim, {{a.x, a.ldx}}), all = layout_of<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.out, a.ldo}});
  const bool hidden = a.relu || a.drop.on;
  bool done;
  if (!all.vec) done = hidden ? by_width<T, kForward>(l.vectors, NormForward<T, true, kMoved>{a, stream}) : by_width<T, kForward>(l.vectors, NormForward<T, false, kMoved>{a, stream});
  else if (l.edge) done = hidden ? by_width<T, kForward>(l.vectors, NormForward<T, true, kEdges>{a, stream}) : by_width<T, kForward>(l.vectors, NormForward<T, false, kEdges>{a, stream});
  else done = hidden ? by_width<T, kForward>(l.vectors, NormForward<T, true, kWhole>{a, stream}) : by_width<T, kForward>(l.vectors, NormForward<T, false, kWhole>{a, stream});
  if (!done) norm_forward_plain<T><<<clamp_blocks(a.rows, kSMs * 8), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

template <class T>
cudaError_t launch_norm_backward(const NormArgs& given, cudaStream_t stream) {
  const NormArgs a = one_row(given);
  int blocks = 0;
  bool done = tiled<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.dy, a.lddy}, {a.out, a.ldo}});
  if (done) {
    const RowRunArgs t{a.x, a.dy, a.out, a.weight, a.bias, a.wf32, a.stats, a.partial, a.rows, a.dim, a.eps, a.relu, a.drop};
    const cudaError_t e = tile_launcher(T{})(t, a.relu || a.drop.on ? kNormBackwardHidden : kNormBackward, stream, &blocks);
    if (e != cudaSuccess) return e;
  }
  const Layout l = layout_of<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.dy, a.lddy}}), all = layout_of<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.dy, a.lddy}, {a.out, a.ldo}});
  const bool hidden = a.relu || a.drop.on;
  if (!done && l.vec) {
    if (!all.vec) done = hidden ? by_width<T, kBackwardHidden>(l.vectors, NormBackward<T, true, kMoved>{a, stream, &blocks}) : by_width<T, kBackward>(l.vectors, NormBackward<T, false, kMoved>{a, stream, &blocks});
    else if (l.edge) done = hidden ? by_width<T, kBackwardHidden>(l.vectors, NormBackward<T, true, kEdges>{a, stream, &blocks}) : by_width<T, kBackward>(l.vectors, NormBackward<T, false, kEdges>{a, stream, &blocks});
    else done = hidden ? by_width<T, kBackwardHidden>(l.vectors, NormBackward<T, true, kWhole>{a, stream, &blocks}) : by_width<T, kBackward>(l.vectors, NormBackward<T, false, kWhole>{a, stream, &blocks});
  }
  if (!done) {
    if (a.out != nullptr) norm_backward_rows_plain<T><<<clamp_blocks(a.rows, kSMs * 8), 256, 0, stream>>>(a);
    if (a.partial != nullptr) {
      blocks = clamp_blocks((a.rows + 31) / 32, column_blocks_cap(a.rows, a.dim));
      norm_backward_columns_plain<T><<<dim3((a.dim + 127) / 128, blocks), 128, 0, stream>>>(a, (a.rows + blocks - 1) / blocks);
    }
  }
  if (a.partial == nullptr) return cudaGetLastError();
  return launch_join<T>(a.partial, blocks, 2 * (int64_t)a.dim, a.dim, a.dweight, a.dbias, a.wf32, stream);
}

// As many blocks as run at once; a multiple of 8, so that a thread's rows keep their distance to the 16-byte boundaries.
template <class T, bool BACK, bool DRAW, bool EDGE>
int launch_dropout_rows(const DropArgs& a, int groups, int threads, int tiles, int smem, cudaStream_t stream) {
  auto kernel = dropout_rows_kernel<T, BACK, DRAW, EDGE>;
  static const int full = blocks_per_sm(kernel, 256, BACK ? 256 * kVec<T> * 4 : 0);
  int64_t most = (int64_t)kSMs * (full * 256 / threads) / tiles;
  if (a.partial != nullptr) most = std::min<int64_t>(most, column_blocks_cap(a.rows, a.dim));
  const int n = clamp_blocks((a.rows + groups - 1) / groups, std::max<int64_t>(most, 8));
  const int blocks = n < 8 ? 8 : n / 8 * 8;
  kernel<<<dim3(blocks, tiles), threads, smem, stream>>>(a);
  return blocks;
}

template <class T, bool BACK>
cudaError_t launch_dropout(const DropArgs& given, cudaStream_t stream) {
  DropArgs a = given;
  if (a.rows <= 1) a.ldx = a.ldy = a.ldo = 0;
  constexpr int V = kVec<T>;
  const Layout l = layout_of<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.y, a.ldy}, {a.out, a.ldo}});
  const bool draw = a.drop.on && !(BACK && a.relu);
  const auto whole = [&](const void* p, int64_t ld) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (a.rows == 1 || ld == a.dim));
  };
  if (a.partial == nullptr && a.bias == nullptr && whole(a.x, a.ldx) && whole(a.y, a.ldy) && whole(a.out, a.ldo)) {
    const int64_t n = a.rows * a.dim;
    const int per = BACK && !draw ? 512 : 1024, blocks = (int)std::max<int64_t>(1, (n / V + per - 1) / per);
    if (!draw) dropout_flat_kernel<T, BACK, false, false><<<blocks, 256, 0, stream>>>(a, n);
    else if (a.drop.first % 4 == 0) dropout_flat_kernel<T, BACK, true, false><<<blocks, 256, 0, stream>>>(a, n);
    else dropout_flat_kernel<T, BACK, true, true><<<blocks, 256, 0, stream>>>(a, n);
    return cudaGetLastError();
  }
  const int tiles = (l.vectors + 255) / 256;
  int blocks = 0;
  if (tiled<T>(a.rows, a.dim, {{a.x, a.ldx}, {a.y, a.ldy}, {a.out, a.ldo}})) {
    const RowRunArgs t{a.x, a.y, a.out, nullptr, a.bias, a.bf32, nullptr, a.partial, a.rows, a.dim, 0.0f, a.relu, a.drop};
    const cudaError_t e = tile_launcher(T{})(t, BACK ? kDropBackward : kDropForward, stream, &blocks);
    if (e != cudaSuccess) return e;
  } else if (l.vec && tiles <= 65535) {
    a.lanes = std::min(l.vectors, 256);
    const int groups = 256 / a.lanes, threads = (groups * a.lanes + 31) / 32 * 32;
    const int smem = BACK && a.partial != nullptr ? groups * a.lanes * V * 4 : 0;
    if (draw && l.edge) blocks = launch_dropout_rows<T, BACK, true, true>(a, groups, threads, tiles, smem, stream);
    else if (draw) blocks = launch_dropout_rows<T, BACK, true, false>(a, groups, threads, tiles, smem, stream);
    else if (l.edge) blocks = launch_dropout_rows<T, BACK, false, true>(a, groups, threads, tiles, smem, stream);
    else blocks = launch_dropout_rows<T, BACK, false, false>(a, groups, threads, tiles, smem, stream);
  } else {
    // the sums first: dx may be dy itself
    if (BACK && a.partial != nullptr) {
      blocks = clamp_blocks((a.rows + 31) / 32, column_blocks_cap(a.rows, a.dim));
      dropout_columns_plain<T><<<dim3((a.dim + 127) / 128, blocks), 128, 0, stream>>>(a, (a.rows + blocks - 1) / blocks);
    }
    if (a.out != nullptr) {
      // contiguous, and element i0 of a group lies at a multiple of four elements
      const auto fours = [&](const void* p, int64_t ld) {
        return (a.rows == 1 || ld == a.dim) && (reinterpret_cast<uintptr_t>(p) / sizeof(T) - a.drop.first) % 4 == 0;
      };
      const int even = (fours(a.x, a.ldx) ? 1 : 0) | (fours(a.y, a.ldy) ? 2 : 0) | (fours(a.out, a.ldo) ? 4 : 0);
      const int64_t groups = a.rows * a.dim / 4 + 2;
      dropout_any_kernel<T, BACK><<<(int)((groups + 511) / 512), 256, 0, stream>>>(a, even);
    }
  }
  if (!BACK || a.partial == nullptr) return cudaGetLastError();
  return launch_join<T>(a.partial, blocks, a.dim, 0, nullptr, a.dbias, a.bf32, stream);
}

}  // namespace

template <class T>
constexpr NormLaunchers launchers() {
  return {launch_norm_forward<T>, launch_norm_backward<T>, launch_dropout<T, false>, launch_dropout<T, true>};
}

}  // namespace rof
