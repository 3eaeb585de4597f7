// Layer norm and dropout for contiguous matrices of up to 511 columns whose rows are not whole 16-byte vectors.
//
// Rows like these share their 16-byte vectors with their neighbours, and a thread that owns vectors of one row spends more
// instructions on the row's two ends than on its middle (47 columns in bf16: 35 instructions an element).  But R = 256 / L rows of a
// contiguous matrix (R a multiple of 8) are whole vectors again, whatever the width.  So a block takes R rows at a time as
// one run of bytes: 16-byte asynchronous copies bring the run into shared memory, S - 1 runs ahead; L threads per row work on pairs of
// elements there, leave the results in place of the input; and the run goes back in
// 16-byte stores.  Dropout is decided on the run too, where four neighbours share a call of the generator: the forward
// pass clears what is dropped on the way out, the backward pass in dy on the way in.
//
// Measured, of the measured copy bandwidth: 2449029x47 layer norm fp32 160 us forward, 242 us back (88 %: HBM), bf16 107 and 148 us (66 and
// 72 %); with ReLU and dropout fp32 203 and 281 us (70 and 76 %), bf16 223 and 254 us (32 and 42 %).  The forward pass in 16 bits keeps
// 71 % of the issue slots busy (24 instructions an element); the others are short of both limits, with 24 to 34 % of the warps and two
// barriers a tile.  L and E follow the width: the fewest lanes whose registers hold the row (half as many elements a thread: 205 us
// instead of 171 forward in bf16).
#pragma once
#include <type_traits>

#include "norm_device.cuh"

namespace rof {
namespace {

constexpr int kTileSlots = 3;

// two neighbouring elements of shared memory, the first at an even place
__device__ __forceinline__ float2 pair_load(const float* p) { return *reinterpret_cast<const float2*>(p); }
__device__ __forceinline__ float2 pair_load(const __nv_bfloat16* p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p)); }
__device__ __forceinline__ float2 pair_load(const __half* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }

// clears the dropped ones of a vector's elements, whose words are w[0 .. V)
template <class T>
__device__ __forceinline__ void clear_dropped(const Drop& d, const uint32_t* w, uint4& raw) {
  uint32_t* word = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    if constexpr (sizeof(T) == 4) word[t] = w[t] > d.last ? word[t] : 0u;
    else word[t] &= (w[2 * t] > d.last ? 0x0000ffffu : 0u) | (w[2 * t + 1] > d.last ? 0xffff0000u : 0u);
  }
}

// Blocks per SM that the register allocation aims at: as many as spill at most 16 bytes.
template <int MODE, int E>
constexpr int tile_blocks() {
  return MODE == kNormBackwardHidden ? (E <= 4 ? 3 : 2) : MODE == kNormBackward ? (E <= 8 ? 3 : 2) : MODE == kNormForwardHidden ? (E <= 12 ? 3 : 2) : (E <= 8 ? 4 : 3);
}

// E elements per thread.  Pair j of lane i holds columns c, c + 1 with c = 2 (i + L j) - s: s = 1 for the odd rows of an odd width (ODD),
// which begin in the middle of a pair; a row's place in its tile is the same in all tiles, so a thread's columns never change.  One
// element of one pair of a row then belongs to the neighbouring row: the first of pair 0 (s = 1) or the second of the
// last pair (s = 0).  It is read as zero and not written.  FEWEST: the rows have more columns than this, so the pairs in front
// of it need no comparison.
template <class T, bool ODD, int L, int E, int FEWEST, int MODE>
__global__ void __launch_bounds__(256, tile_blocks<MODE, E>()) norm_tile_kernel(const __grid_constant__ RowRunArgs a) {
  constexpr int V = kVec<T>, S = kTileSlots, P = E / 2, R = 256 / L;
  constexpr int M = (E * (int)sizeof(T) + 15) / 16;  // vectors of a tile per thread, at most
  constexpr bool kNorm = MODE <= kNormBackwardHidden, kBack = MODE == kNormBackward || MODE == kNormBackwardHidden || MODE == kDropBackward;
  constexpr bool kHidden = MODE == kNormForwardHidden || MODE == kNormBackwardHidden;
  constexpr bool kWeight = kNorm, kBias = MODE != kNormBackward && MODE != kDropBackward;
  constexpr int kSure = (FEWEST + 1) / 2 / L;     // pairs 0 .. kSure - 1 lie in the row (but for the first element of pair 0)
  extern __shared__ uint4 tile_memory[];
  const Group<L> g;
  const int dim = a.dim, tid = threadIdx.x;
  const int vectors = R * dim / V;                  // of a whole tile
  const bool second = kBack && a.b != nullptr;
  // this block's tiles, whole ones first
  const int64_t all_tiles = (a.rows + R - 1) / R, whole_tiles = a.rows / R;
  const int tiles = blockIdx.x < all_tiles ? (int)((all_tiles - blockIdx.x + gridDim.x - 1) / gridDim.x) : 0;
  const int whole = blockIdx.x < whole_tiles ? (int)((whole_tiles - blockIdx.x + gridDim.x - 1) / gridDim.x) : 0;
  const int last = (int)(a.rows - whole_tiles * R) * dim;        // elements of the matrix's last tile, where it is not whole
  constexpr int kSureM = R * (FEWEST + 1) / V / 256;             // every thread has this many vectors of a tile
  const uint64_t step = step_of(a.drop);
  const bool draw_in = (MODE == kNormBackwardHidden && a.drop.on) || (MODE == kDropBackward && a.drop.on && !a.relu);
  const bool draw_out = (MODE == kNormForwardHidden || MODE == kDropForward) && a.drop.on;
  const float inv = 1.0f / (float)dim;
  const int s = ODD ? (g.index * dim) & 1 : 0;
  const int c0 = 2 * g.lane - s;                    // the column of pair j is c0 + 2 L j

  const int slot_bytes = (kBack ? 2 : 1) * vectors * 16;
  char* const memory = reinterpret_cast<char*>(tile_memory);
  const int64_t tile0 = (int64_t)blockIdx.x * (R * dim), tile_step = (int64_t)gridDim.x * (R * dim);   // in elements
  const T* from_a = reinterpret_cast<const T*>(a.a) + tile0 + tid * V;
  const T* from_b = reinterpret_cast<const T*>(a.b) + tile0 + tid * V;
  const auto mine = [&](int m, int n) { return m < kSureM || m * 256 + tid < n; };
  // brings the next tile, the i-th, into the slot at byte `at`; what lies behind the matrix is zero
  const auto fetch = [&](int i, int at) {
    uint4* pa = reinterpret_cast<uint4*>(memory + at) + tid;
    uint4* pb = pa + vectors;
    if (i < whole) {
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (mine(m, vectors)) {
          copy_async(pa + m * 256, from_a + m * 256 * V, 16);
          if (second) copy_async(pb + m * 256, from_b + m * 256 * V, 16);
        }
    } else {
#pragma unroll 1
      for (int m = 0; m < M; ++m) {
        const int bytes = min(16, (last - (m * 256 + tid) * V) * (int)sizeof(T));
        if (bytes > 0) {
          copy_async(pa + m * 256, from_a + m * 256 * V, bytes);
          if (second) copy_async(pb + m * 256, from_b + m * 256 * V, bytes);
        }
      }
    }
    from_a += tile_step;
    from_b += tile_step;
  };
  // a row's pairs in shared memory
  const auto read = [&](const T* row, float2 (&v)[P]) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = c0 + 2 * L * j;
      if (j < kSure) {
        v[j] = pair_load(row + c);
      } else {
        v[j] = c < dim ? pair_load(row + c) : both(0.0f);
        if (ODD && c + 1 >= dim) v[j].y = 0.0f;
      }
    }
    if (ODD && c0 < 0) v[0].x = 0.0f;
  };
  constexpr bool kMark = MODE == kDropForward && sizeof(T) == 2;   // the ReLU follows the rounding
  const auto write = [&](T* row, int j, float2 v) {
    const int c = c0 + 2 * L * j;
    if constexpr (kMark) {
      if (a.relu) {
        alignas(4) T two[2];
        pack_two(two, v);
        uint32_t* pair = reinterpret_cast<uint32_t*>(two);
        *pair = relu_marked<T>(*pair);
        if (ODD && j == 0 && c < 0) row[0] = two[1];
        else if (j < kSure || c + 1 < dim) *reinterpret_cast<uint32_t*>(row + c) = *pair;
        else if (ODD && c < dim) row[c] = two[0];
        return;
      }
    }
    if (ODD && j == 0 && c < 0) row[0] = from_float<T>(v.y);
    else if (j < kSure || c + 1 < dim) pack_two(row + c, v);
    else if (ODD && c < dim) row[c] = from_float<T>(v.x);
  };

#pragma unroll
  for (int i = 0; i < S - 1; ++i) {
    if (i < tiles) fetch(i, i * slot_bytes);
    copy_commit();
  }
  float2* stats = a.stats + g.first;
  const int64_t row_step = (int64_t)gridDim.x * R;
  float2 st_next = both(0.0f);
  if constexpr (kNorm && kBack) {
    if (g.first < a.rows) st_next = *stats;
  }
  float2 w[kWeight ? P : 1], b[kBias ? P : 1], aw[kNorm && kBack ? P : 1], ab[kBack ? P : 1];
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = c0 + 2 * L * j, d = c + 1;
    if constexpr (kWeight) {
      w[j].x = a.weight != nullptr && (unsigned)c < (unsigned)dim ? vector_at<T>(a.weight, a.f32, c) : 1.0f;
      w[j].y = a.weight != nullptr && d < dim ? vector_at<T>(a.weight, a.f32, d) : 1.0f;
    }
    if constexpr (kBias) {
      b[j].x = a.bias != nullptr && (unsigned)c < (unsigned)dim ? vector_at<T>(a.bias, a.f32, c) : 0.0f;
      b[j].y = a.bias != nullptr && d < dim ? vector_at<T>(a.bias, a.f32, d) : 0.0f;
    }
    if constexpr (kNorm && kBack) aw[j] = both(0.0f);
    if constexpr (kBack) ab[j] = both(0.0f);
  }

  int at = 0, next = (S - 1) * slot_bytes;
  T* out = reinterpret_cast<T*>(a.out) + tile0 + tid * V;
  int64_t e = a.drop.first + tile0 + tid * V;
  for (int i = 0; i < tiles; ++i) {
    const bool live = i < whole || g.index * dim < last;
    const float2 st = st_next;
    if constexpr (kNorm && kBack) {
      if (i + 1 < whole || (i + 1 < tiles && g.index * dim < last)) st_next = stats[row_step];
    }
    if constexpr (MODE == kNormBackwardHidden || MODE == kDropBackward) {
      if (draw_in) {                                // on the vectors that this thread copied itself
        uint32_t words[M * V];
        draw_words<M, V, true>(a.drop, step, e, 256 * V, words);
        copy_wait<S - 2>();
        uint4* p = reinterpret_cast<uint4*>(memory + at) + (kNorm ? vectors : 0) + tid;
#pragma unroll
        for (int m = 0; m < M; ++m) {
          if (mine(m, vectors)) {
            uint4 raw = p[m * 256];
            clear_dropped<T>(a.drop, words + m * V, raw);
            p[m * 256] = raw;
          }
        }
      }
    }
    copy_wait<S - 2>();
    __syncthreads();                                // the tile is complete, and the slot before it is free
    if (i + S - 1 < tiles) fetch(i + S - 1, next);
    copy_commit();

    T* pa = reinterpret_cast<T*>(memory + at) + g.index * dim;
    const T* pb = reinterpret_cast<const T*>(memory + at + vectors * 16) + g.index * dim;
    if (live) {
      float2 v[P];
      read(pa, v);
      if constexpr (MODE == kNormForward || MODE == kNormForwardHidden) {
        float2 sum = both(0.0f), dev1 = both(0.0f), dev2 = both(0.0f);
#pragma unroll
        for (int j = 0; j < P; ++j) sum = __fadd2_rn(sum, v[j]);
        float mean = g.sum(sum.x + sum.y, nullptr) * inv;
        float2 minus = both(-mean);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const int c = c0 + 2 * L * j;
          float2 x = __fadd2_rn(v[j], minus);
          if (j >= kSure) x = make_float2(c < dim ? x.x : 0.0f, c + 1 < dim ? x.y : 0.0f);
          if (ODD && j == 0 && c0 < 0) x.x = 0.0f;
          dev1 = __fadd2_rn(dev1, x);
          dev2 = __ffma2_rn(x, x, dev2);
        }
        const float2 dev = g.sum(make_float2(dev1.x + dev1.y, dev2.x + dev2.y), nullptr);
        const float off = dev.x * inv;
        mean += off;
        minus = both(-mean);
        const float rstd = rsqrt_of(variance_of(dev.y * inv, off) + a.eps);
        if (a.stats != nullptr && g.lane == 0) *stats = make_float2(mean, rstd);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          float2 z = __ffma2_rn(__fmul2_rn(__fadd2_rn(v[j], minus), both(rstd)), w[j], b[j]);
          if constexpr (kHidden) {
            if (a.relu) z = make_float2(relu_of(z.x), relu_of(z.y));
            z = __fmul2_rn(z, both(a.drop.scale));
          }
          write(pa, j, z);
        }
      } else if constexpr (kNorm) {
        const float2 minus = both(-st.x), rstd = both(st.y);
        float2 gr[P], s1 = both(0.0f), s2 = both(0.0f);
        read(pb, gr);
#pragma unroll
        for (int j = 0; j < P; ++j) {
          // (what lies outside the row has x = dy = 0 and adds nothing anywhere)
          float2 dz = gr[j];
          v[j] = __fmul2_rn(__fadd2_rn(v[j], minus), rstd);
          if constexpr (kHidden) {
            dz = __fmul2_rn(dz, both(a.drop.scale));
            if (a.relu) {
              const float2 z = __ffma2_rn(v[j], w[j], b[j]);
              dz = make_float2(z.x <= 0.0f ? 0.0f : dz.x, z.y <= 0.0f ? 0.0f : dz.y);
            }
          }
          aw[j] = __ffma2_rn(dz, v[j], aw[j]);
          ab[j] = __fadd2_rn(ab[j], dz);
          gr[j] = __fmul2_rn(dz, w[j]);
          s1 = __fadd2_rn(s1, gr[j]);
          s2 = __ffma2_rn(gr[j], v[j], s2);
        }
        if (a.out != nullptr) {
          const float2 sums = g.sum(make_float2(s1.x + s1.y, s2.x + s2.y), nullptr);
          const float2 c1 = both(-sums.x * inv), c2 = both(-sums.y * inv);
#pragma unroll
          for (int j = 0; j < P; ++j) write(pa, j, __fmul2_rn(__fadd2_rn(gr[j], __ffma2_rn(v[j], c2, c1)), rstd));
        }
      } else {
        if constexpr (kBack) {
          if (second) {
            float2 y[P];
            read(pb, y);
#pragma unroll
            for (int j = 0; j < P; ++j) v[j] = make_float2(passed_of(y[j].x, v[j].x), passed_of(y[j].y, v[j].y));
          }
        } else {
#pragma unroll
          for (int j = 0; j < P; ++j) v[j] = __fadd2_rn(v[j], b[j]);
          if (!kMark && a.relu) {
#pragma unroll
            for (int j = 0; j < P; ++j) v[j] = make_float2(relu_of(v[j].x), relu_of(v[j].y));
          }
        }
        const float least = kMark && a.relu ? -kLeast : -0.0f;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          v[j] = __ffma2_rn(v[j], both(a.drop.scale), both(least));
          if constexpr (kBack) ab[j] = __fadd2_rn(ab[j], v[j]);
          write(pa, j, v[j]);
        }
      }
    }
    if (a.out != nullptr) {
      uint32_t words[kBack ? 1 : M * V];
      if constexpr (!kBack) {
        if (draw_out) draw_words<M, V, true>(a.drop, step, e, 256 * V, words);
      }
      __syncthreads();                              // the results are complete
      const uint4* p = reinterpret_cast<const uint4*>(memory + at) + tid;
      const int n = i < whole ? vectors : last / V;
#pragma unroll
      for (int m = 0; m < M; ++m)
        if (i < whole ? mine(m, vectors) : m * 256 + tid < n) {
          uint4 raw = p[m * 256];
          if constexpr (!kBack) {
            if (draw_out) clear_dropped<T>(a.drop, words + m * V, raw);
          }
          *reinterpret_cast<uint4*>(out + m * 256 * V) = raw;
        }
      // the matrix's last elements that fill no vector
      if (i >= whole && tid < last - n * V) {
        const int64_t off = n * V + tid - tid * V;
        const bool keep = kBack || !draw_out || kept(a.drop, step, e + off);
        out[off] = keep ? reinterpret_cast<const T*>(memory + at)[n * V + tid] : from_float<T>(0.0f);
      }
      out += tile_step;
    }
    e += tile_step;
    if constexpr (kNorm) stats += row_step;
    next = at;
    at = at == (S - 1) * slot_bytes ? 0 : at + slot_bytes;
  }

  if constexpr (kBack) {
    if (a.partial == nullptr) return;
    copy_wait<0>();
    float* sums = reinterpret_cast<float*>(tile_memory);
    float* p = a.partial + (int64_t)blockIdx.x * (kNorm ? 2 : 1) * dim;
#pragma unroll
    for (int pass = kNorm ? 0 : 1; pass < 2; ++pass) {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float2 v = pass == 0 ? aw[kNorm ? j : 0] : ab[j];
        const int c = c0 + 2 * L * j;
        if ((unsigned)c < (unsigned)dim) sums[g.index * dim + c] = v.x;
        if (c + 1 < dim) sums[g.index * dim + c + 1] = v.y;
      }
      __syncthreads();
      for (int c = tid; c < dim; c += 256) {
        float sum = 0.0f;
#pragma unroll 8
        for (int i = 0; i < R; ++i) sum += sums[i * dim + c];
        p[(kNorm ? pass : 0) * dim + c] = sum;
      }
    }
  }
}

template <class T, bool ODD, int MODE>
struct TileLaunch {
  const RowRunArgs& a;
  cudaStream_t stream;
  int* blocks;
  template <int L, int E, int FEWEST>
  void run() const {
    auto kernel = norm_tile_kernel<T, ODD, L, E, FEWEST, MODE>;
    constexpr int R = 256 / L, streams = MODE == kNormBackward || MODE == kNormBackwardHidden || MODE == kDropBackward ? 2 : 1;
    constexpr int most_smem = kTileSlots * streams * R * L * E * (int)sizeof(T);
    const int smem = kTileSlots * streams * R * a.dim * (int)sizeof(T);
    static std::atomic<uint64_t> seen{0};
    allow_smem(kernel, most_smem, seen);
    static const int full = blocks_per_sm(kernel, 256, most_smem);
    int64_t most = (int64_t)kSMs * full;
    if (a.partial != nullptr) most = std::min<int64_t>(most, column_blocks_cap(a.rows, a.dim));
    const int n = clamp_blocks((a.rows + R - 1) / R, most);
    kernel<<<n, 256, smem, stream>>>(a);
    if (blocks != nullptr) *blocks = n;
  }
  void by_columns() const {
    const int d = a.dim;
    if (d <= 15) run<4, 4, 0>();
    else if (d <= 31) run<4, 8, 15>();
    else if (d <= 47) run<4, 12, 31>();
    else if (d <= 63) run<4, 16, 47>();
    else if (d <= 95) run<8, 12, 63>();
    else if (d <= 127) run<8, 16, 95>();
    else if (d <= 191) run<16, 12, 127>();
    else if (d <= 255) run<16, 16, 191>();
    else if (d <= 383) run<32, 12, 255>();
    else run<32, 16, 383>();
  }
};

template <class T>
cudaError_t launch_tile(const RowRunArgs& a, int mode, cudaStream_t stream, int* blocks) {
  const auto go = [&](auto odd) {
    constexpr bool ODD = decltype(odd)::value;
    switch (mode) {
      case kNormForward: TileLaunch<T, ODD, kNormForward>{a, stream, blocks}.by_columns(); break;
      case kNormForwardHidden: TileLaunch<T, ODD, kNormForwardHidden>{a, stream, blocks}.by_columns(); break;
      case kNormBackward: TileLaunch<T, ODD, kNormBackward>{a, stream, blocks}.by_columns(); break;
      case kNormBackwardHidden: TileLaunch<T, ODD, kNormBackwardHidden>{a, stream, blocks}.by_columns(); break;
      case kDropForward: TileLaunch<T, ODD, kDropForward>{a, stream, blocks}.by_columns(); break;
      default: TileLaunch<T, ODD, kDropBackward>{a, stream, blocks}.by_columns(); break;
    }
  };
  if (a.dim % 2) go(std::true_type{});
  else go(std::false_type{});
  return cudaGetLastError();
}

}  // namespace
}  // namespace rof
