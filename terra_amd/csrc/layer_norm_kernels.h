// The kernels of layer_norm.h for one pair of types of x and y.
#pragma once

#include "layer_norm.h"

namespace terra {
namespace {

template <int DTX, int DTY>
constexpr int norm_pieces() { return DTX == TERRA_DTYPE_F32 || DTY == TERRA_DTYPE_F32 ? 4 : 8; }

// ---- rows held in registers ------------------------------------------------------

// The next rows are fetched before the ones at hand are worked on.
template <int DTX, int DTY, int kG, int kK, bool kVec, bool kPairs>
__global__ __launch_bounds__(tail_threads(kG)) void norm_kernel(const NormArgs a) {
  constexpr int kGroups = tail_threads(kG) / kG, kYB = ChunkElt<DTY>::kBytes, kP = norm_pieces<DTX, DTY>();
  using Param = NormParam<kG, kK, kP>;
  __shared__ typename RowSum<kG>::Shared s_red;
  __shared__ typename Param::Shared s_w, s_b;
  const int group = threadIdx.x / kG, C = a.C;
  const RowLanes<kG, kK, kP> at = {(int)(threadIdx.x % kG), C};
  RowSum<kG> sum(&s_red);
  const bool full = C == kG * kK * kChunkCols;  // every lane has columns
  Param w(&s_w), b(&s_b);
  struct Row { RowChunk<DTX> x[kK]; };
  auto fetch = [&](uint32_t base) {  // a row past the end re-reads the last one
    Row q;
    const uint32_t row = base + group;
    const uint8_t* xp = a.row(row < a.rows ? row : a.rows - 1);
#pragma unroll
    for (int k = 0; k < kK; ++k) q.x[k] = at.template load<DTX, kVec, kPairs>(xp, k);
    return q;
  };
  const uint32_t step = gridDim.x * kGroups;
  uint32_t base = blockIdx.x * kGroups;
  Row ahead = fetch(base);
  w.template fill<kVec>(at, a.w, a.param_dtype, 1.f);
  b.template fill<kVec>(at, a.b, a.param_dtype, 0.f);
  if constexpr (Param::kLds) RowSum<kG>::lds_sync();
  for (; base < a.rows; base += step) {
    // Parameters in LDS are read in each turn: over the loop they would take the registers of other waves.
    if constexpr (Param::kLds) asm volatile("" ::: "memory");
    const Row q = ahead;
    if (base + step < a.rows) ahead = fetch(base + step);
    const uint32_t r = base + group;
    const bool live = r < a.rows;
    float v[kK][kChunkCols], mean;
#pragma unroll
    for (int k = 0; k < kK; ++k) at.template values<DTX, kVec>(q.x[k], k, true, full, v[k]);
    const float rs = norm_row<kG, kK, kP, kVec>(v, a.layer, a.eps, a.inv_c, at, sum, mean);
    if (a.statistics != nullptr && live && at.lane == 0) a.statistics[r] = make_float2(mean, rs);
    const __amdgpu_buffer_rsrc_t out =
        buffer_rsrc(a.y + (int64_t)base * C * kYB, min(a.rows - base, (uint32_t)kGroups) * (uint32_t)(C * kYB));
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      float wv[kChunkCols], bv[kChunkCols];
      w.get(k, at, wv);
      b.get(k, at, bv);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[k][j] = fmaf(v[k][j], wv[j], bv[j]);
      if (live) at.template store<DTY, kVec>(v[k], out, (uint32_t)(group * C) * kYB, a.y + (int64_t)r * C * kYB, k);
    }
  }
}

// Each lane keeps the sums of its columns over the rows that it takes.
template <int DTX, int DTY, int kG, int kK, bool kVec, bool kPairs>
__global__ __launch_bounds__(tail_threads(kG)) void norm_bwd_kernel(const NormArgs a) {
  constexpr int kThreads = tail_threads(kG), kGroups = kThreads / kG, kCols = kG * kK * kChunkCols;
  constexpr int kXB = ChunkElt<DTX>::kBytes, kYB = ChunkElt<DTY>::kBytes, kP = norm_pieces<DTX, DTY>();
  using Param = NormParam<kG, kK, kP>;
  __shared__ typename RowSum<kG>::Shared s_red;
  __shared__ typename Param::Shared s_w;
  __shared__ __attribute__((aligned(16))) float s_acc[kGroups > 1 ? kGroups * kCols : 1];
  const int group = threadIdx.x / kG, C = a.C;
  const RowLanes<kG, kK, kP> at = {(int)(threadIdx.x % kG), C};
  RowSum<kG> sum(&s_red);
  const bool full = C == kG * kK * kChunkCols;
  Param weight(&s_w);
  weight.template fill<kVec>(at, a.w, a.param_dtype, 1.f);
  if constexpr (Param::kLds) RowSum<kG>::lds_sync();
  float acc_w[kK][kChunkCols] = {}, acc_b[kK][kChunkCols] = {};
  for (uint32_t base = blockIdx.x * kGroups; base < a.rows; base += gridDim.x * kGroups) {
    if constexpr (Param::kLds) asm volatile("" ::: "memory");
    const uint32_t row = base + group;
    const bool live = row < a.rows;
    const uint32_t r = live ? row : a.rows - 1;  // a row past the end re-reads the last one
    RowChunk<DTX> xq[kK];
    RowChunk<DTY> dq[kK];
    const uint8_t *xp = a.row(r), *dp = a.dy + (int64_t)r * C * kYB;
    const float2 st = a.statistics[r];
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      xq[k] = at.template load<DTX, kVec, kPairs>(xp, k);
      dq[k] = at.template load<DTY, kVec, kPairs>(dp, k);
    }
    float v[kK][kChunkCols], g[kK][kChunkCols], s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      float w[kChunkCols];
      weight.get(k, at, w);
      at.template values<DTX, kVec>(xq[k], k, true, true, v[k]);  // absent columns have no gradient
      at.template values<DTY, kVec>(dq[k], k, true, full, g[k]);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[k][j] = (v[k][j] - st.x) * st.y;
      if (live)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          acc_w[k][j] = fmaf(g[k][j], v[k][j], acc_w[k][j]);
          acc_b[k][j] += g[k][j];
        }
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        g[k][j] *= w[j];
        s0 += g[k][j];
        s1 = fmaf(g[k][j], v[k][j], s1);
      }
    }
    if (a.dx == nullptr) continue;
    sum.two(s0, s1);
    s0 = a.layer ? s0 * a.inv_c : 0.f;
    s1 *= a.inv_c;
    const __amdgpu_buffer_rsrc_t out =
        buffer_rsrc(a.dx + (int64_t)base * C * kXB, min(a.rows - base, (uint32_t)kGroups) * (uint32_t)(C * kXB));
#pragma unroll
    for (int k = 0; k < kK; ++k) {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) g[k][j] = st.y * fmaf(-s1, v[k][j], g[k][j] - s0);
      if (live) at.template store<DTX, kVec>(g[k], out, (uint32_t)(group * C) * kXB, a.dx + (int64_t)r * C * kXB, k);
    }
  }
  if (a.partial == nullptr) return;
  float* const mine = a.partial + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float (&acc)[kK][kChunkCols] = which == 0 ? acc_w : acc_b;
    if constexpr (kGroups > 1) {
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        *reinterpret_cast<float4*>(&s_acc[group * kCols + at.base(k, 0)]) = make_float4(acc[k][0], acc[k][1], acc[k][2], acc[k][3]);
        *reinterpret_cast<float4*>(&s_acc[group * kCols + at.base(k, 1)]) = make_float4(acc[k][4], acc[k][5], acc[k][6], acc[k][7]);
      }
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += kThreads) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) t += s_acc[i * kCols + c];
        mine[which * C + c] = t;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const int c = at.base(k, j >> 2) + (j & 3);
          if (c < C) mine[which * C + c] = acc[k][j];
        }
    }
  }
}

// ---- packed rows that are not whole aligned chunks -------------------------------
// The rows of a packed tensor that begins aligned, read and written by the aligned
// chunks of the tensor: a row's first and last one may hold columns of its neighbours too.  Row r begins
// r C modulo the chunk into one, so rows eight apart stand alike in their chunks: a group takes such rows alone, and
// each lane's columns, parameters and sums are the same for all of them.  (One column at a time a 16-bit row takes
// twice as long.)
template <int kG, int kK, int kP>
struct FlatLanes {
  int lane, C, shift;    // columns that the first chunk holds of the row before
  int64_t elements;      // of the tensor

  __device__ __forceinline__ int base(int k, int half) const {  // the column of a half's first value, from -shift on
    return (kP == 8 ? (lane + kG * k) * 8 + 4 * half : (lane + kG * (2 * k + half)) * 4) - shift;
  }
  __device__ __forceinline__ bool has(int k, int j) const { return (unsigned)(base(k, j >> 2) + (j & 3)) < (unsigned)C; }

  __device__ __forceinline__ void param(const void* p, int dtype, float none, float (&f)[kK][kChunkCols]) const {
    with_param(p, dtype, none, [&](auto load) {
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const float v = load(has(k, j) ? base(k, j >> 2) + (j & 3) : 0);
          f[k][j] = has(k, j) ? v : 0.f;
        }
    });
  }
  // kN values from element `at` of the tensor on, as words.  kInside: all of them are there.
  template <int DT, int kN, bool kInside>
  __device__ __forceinline__ void piece(const uint8_t* tensor, int64_t at, uint32_t* w) const {
    constexpr int kB = ChunkElt<DT>::kBytes, kWords = kN * kB / 4;
    typedef uint32_t Vec __attribute__((ext_vector_type(kWords)));
    if constexpr (kInside) {
      const Vec v = *reinterpret_cast<const Vec*>(tensor + at * kB);
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (kB == 4) {
          w[i] = at + i < elements ? reinterpret_cast<const uint32_t*>(tensor)[at + i] : 0u;
        } else {
          const uint16_t* h = reinterpret_cast<const uint16_t*>(tensor);
          w[i] = (at + 2 * i < elements ? (uint32_t)h[at + 2 * i] : 0u) | (at + 2 * i + 1 < elements ? (uint32_t)h[at + 2 * i + 1] << 16 : 0u);
        }
      }
    }
  }
  template <int DT, bool kInside>
  __device__ __forceinline__ void load(const uint8_t* tensor, int64_t first, RowChunk<DT> (&r)[kK]) const {
    constexpr int kHalf = ChunkElt<DT>::kBytes;  // words of four values
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      uint32_t w[2 * kHalf];
#pragma unroll
      for (int h = 0; h < (kP == 8 ? 1 : 2); ++h) {
        const int col = base(k, h);  // an absent piece reads the row's first
        piece<DT, kP, kInside>(tensor, first + (col < C ? col : -shift), w + h * kHalf);
      }
#pragma unroll
      for (int i = 0; i < RowChunk<DT>::kWords; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) r[k].q[i][j] = w[4 * i + j];
    }
  }
  // The row whose first element is `first`.  Its last chunk may go past the end of the tensor: tested once for the wave.
  template <int DT>
  __device__ __forceinline__ void load(const uint8_t* tensor, int64_t first, RowChunk<DT> (&r)[kK]) const {
    if (__builtin_amdgcn_ballot_w64(first + C + kP - 1 > elements) == 0) load<DT, true>(tensor, first, r);
    else load<DT, false>(tensor, first, r);
  }
  // Its values in fp32, zeros in absent columns.
  template <int DT>
  __device__ __forceinline__ void values(const RowChunk<DT>& r, int k, float (&f)[kChunkCols]) const {
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) f[j] = has(k, j) ? chunk_value<DT>(r, j) : 0.f;
  }
  template <int DT>
  __device__ __forceinline__ void store_four(const float* f, uint8_t* tensor, int64_t first, int col) const {
    constexpr int kB = ChunkElt<DT>::kBytes;
    uint8_t* p = tensor + (first + col) * kB;
    if (col >= 0 && col + 4 <= C) {
      if constexpr (kB == 4)
        *reinterpret_cast<stream_u32x4*>(p) =
            stream_u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
      else
        *reinterpret_cast<stream_u32x2*>(p) = stream_u32x2{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3])};
    } else if (col + 4 > 0 && col < C) {
      if constexpr (kB == 4) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if ((unsigned)(col + j) < (unsigned)C) reinterpret_cast<float*>(p)[j] = f[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {  // by pairs, which stand aligned
          const bool lo = (unsigned)(col + j) < (unsigned)C, hi = (unsigned)(col + j + 1) < (unsigned)C;
          const uint32_t w = pack2<DT>(f[j], f[j + 1]);
          if (lo && hi) reinterpret_cast<uint32_t*>(p)[j / 2] = w;
          else if (lo) reinterpret_cast<uint16_t*>(p)[j] = (uint16_t)w;
          else if (hi) reinterpret_cast<uint16_t*>(p)[j + 1] = (uint16_t)(w >> 16);
        }
      }
    }
  }
  template <int DT>
  __device__ __forceinline__ void store(const float (&f)[kChunkCols], uint8_t* tensor, int64_t first, int k) const {
    if constexpr (kP == 8) {
      const int col = base(k, 0);
      if (col >= 0 && col + 8 <= C) {
        *reinterpret_cast<stream_u32x4*>(tensor + (first + col) * 2) =
            stream_u32x4{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]), pack2<DT>(f[6], f[7])};
        return;
      }
    }
    store_four<DT>(f, tensor, first, base(k, 0));
    store_four<DT>(f + 4, tensor, first, base(k, 1));
  }
};

template <int DTX, int DTY, int kG, int kK>
__global__ __launch_bounds__(tail_threads(kG)) void norm_flat_kernel(const NormArgs a) {
  constexpr int kGroups = tail_threads(kG) / kG, kP = norm_pieces<DTX, DTY>();
  __shared__ typename RowSum<kG>::Shared s_red;
  const int group = threadIdx.x / kG, C = a.C;
  const uint32_t step = gridDim.x * kGroups, row0 = blockIdx.x * kGroups + group;  // step: a multiple of 8
  const uint32_t own = row0 < a.rows ? row0 : 0;  // what a group reads where it has no row
  const FlatLanes<kG, kK, kP> at = {(int)(threadIdx.x % kG), C, (int)(((int64_t)own * C) & (kP - 1)), (int64_t)a.rows * C};
  RowSum<kG> sum(&s_red);
  struct Row { RowChunk<DTX> x[kK]; };
  auto fetch = [&](uint32_t r) {
    Row q;
    const int64_t first = (int64_t)(r < a.rows ? r : own) * C;
    at.template load<DTX>(a.x, first, q.x);
    return q;
  };
  Row ahead = fetch(row0);
  float w[kK][kChunkCols], b[kK][kChunkCols];
  at.param(a.w, a.param_dtype, 1.f, w);
  at.param(a.b, a.param_dtype, 0.f, b);
  // All groups of a workgroup go round as often as its first, whose rows are the earliest.
  for (uint32_t r = row0; r - group < a.rows; r += step) {
    const Row q = ahead;
    if (r - group + step < a.rows) ahead = fetch(r + step);
    const bool live = r < a.rows;
    float v[kK][kChunkCols], mean = 0.f, s = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      at.template values<DTX>(q.x[k], k, v[k]);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) s += v[k][j];
    }
    if (a.layer) mean = sum.one(s) * a.inv_c;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        v[k][j] -= at.has(k, j) ? mean : 0.f;
        s2 = fmaf(v[k][j], v[k][j], s2);
      }
    const float rs = rsqrtf(sum.one(s2) * a.inv_c + a.eps);
    if (a.statistics != nullptr && live && at.lane == 0) a.statistics[r] = make_float2(mean, rs);
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[k][j] = fmaf(v[k][j] * rs, w[k][j], b[k][j]);
      at.template store<DTY>(v[k], a.y, (int64_t)r * C, k);
    }
  }
}

template <int DTX, int DTY, int kG, int kK>
__global__ __launch_bounds__(tail_threads(kG)) void norm_flat_bwd_kernel(const NormArgs a) {
  constexpr int kThreads = tail_threads(kG), kGroups = kThreads / kG, kCols = kG * kK * kChunkCols;
  constexpr int kP = norm_pieces<DTX, DTY>();
  __shared__ typename RowSum<kG>::Shared s_red;
  __shared__ float s_acc[kGroups > 1 ? kGroups * kCols : 1];
  const int group = threadIdx.x / kG, C = a.C;
  const uint32_t step = gridDim.x * kGroups, row0 = blockIdx.x * kGroups + group;
  const uint32_t own = row0 < a.rows ? row0 : 0;
  const FlatLanes<kG, kK, kP> at = {(int)(threadIdx.x % kG), C, (int)(((int64_t)own * C) & (kP - 1)), (int64_t)a.rows * C};
  RowSum<kG> sum(&s_red);
  float w[kK][kChunkCols], acc_w[kK][kChunkCols] = {}, acc_b[kK][kChunkCols] = {};
  at.param(a.w, a.param_dtype, 1.f, w);
  for (uint32_t r = row0; r - group < a.rows; r += step) {
    const bool live = r < a.rows;
    const uint32_t row = live ? r : own;
    const int64_t first = (int64_t)row * C;
    RowChunk<DTX> xq[kK];
    RowChunk<DTY> dq[kK];
    const float2 st = a.statistics[row];
    at.template load<DTX>(a.x, first, xq);
    at.template load<DTY>(a.dy, first, dq);
    float v[kK][kChunkCols], g[kK][kChunkCols], s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      at.template values<DTX>(xq[k], k, v[k]);
      at.template values<DTY>(dq[k], k, g[k]);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[k][j] = (v[k][j] - st.x) * st.y;
      if (live)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          acc_w[k][j] = fmaf(g[k][j], v[k][j], acc_w[k][j]);
          acc_b[k][j] += g[k][j];
        }
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        g[k][j] *= w[k][j];
        s0 += g[k][j];
        s1 = fmaf(g[k][j], v[k][j], s1);
      }
    }
    if (a.dx == nullptr) continue;
    sum.two(s0, s1);
    s0 = a.layer ? s0 * a.inv_c : 0.f;
    s1 *= a.inv_c;
    if (!live) continue;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) g[k][j] = st.y * fmaf(-s1, v[k][j], g[k][j] - s0);
      at.template store<DTX>(g[k], a.dx, first, k);
    }
  }
  if (a.partial == nullptr) return;
  float* const mine = a.partial + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float (&acc)[kK][kChunkCols] = which == 0 ? acc_w : acc_b;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        const int c = at.base(k, j >> 2) + (j & 3);
        if constexpr (kGroups > 1) s_acc[group * kCols + c + at.shift] = acc[k][j];
        else if ((unsigned)c < (unsigned)C) mine[which * C + c] = acc[k][j];
      }
    if constexpr (kGroups > 1) {
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += kThreads) {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < kGroups; ++i)
          t += s_acc[i * kCols + c + (int)(((int64_t)(blockIdx.x * kGroups + i) * C) & (kP - 1))];
        mine[which * C + c] = t;
      }
      __syncthreads();
    }
  }
}

// ---- rows of any width, read again for each pass --------------------------------
// A workgroup a row; what a pass reads again comes from L2.
constexpr int kWideLanes = 512;

template <int DTX, int DTY, bool kVec>
__global__ __launch_bounds__(kWideLanes) void norm_wide_kernel(const NormArgs a) {
  constexpr int kP = norm_pieces<DTX, DTY>(), kYB = ChunkElt<DTY>::kBytes;
  __shared__ typename RowSum<kWideLanes>::Shared s_red;
  RowSum<kWideLanes> sum(&s_red);
  const RowLanes<kWideLanes, 1, kP> at = {(int)threadIdx.x, a.C};
  const int chunks = (a.C + kWideLanes * kChunkCols - 1) / (kWideLanes * kChunkCols);
  for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const uint8_t* row = a.row(r);
    float v[kChunkCols], mean = 0.f, q = 0.f;
    if (a.layer) {
      float s = 0.f;
      for (int k = 0; k < chunks; ++k) {
        at.template values<DTX, kVec>(at.template load<DTX, kVec, false>(row, k), k, true, false, v);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) s += v[j];
      }
      mean = sum.one(s) * a.inv_c;
    }
    for (int k = 0; k < chunks; ++k) {
      at.template values<DTX, kVec>(at.template load<DTX, kVec, false>(row, k), k, true, false, v);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        const float d = at.template has<kVec>(k, j) ? v[j] - mean : 0.f;
        q = fmaf(d, d, q);
      }
    }
    const float rs = rsqrtf(sum.one(q) * a.inv_c + a.eps);
    for (int k = 0; k < chunks; ++k) {
      at.template values<DTX, kVec>(at.template load<DTX, kVec, false>(row, k), k, true, false, v);
      auto column = [&](int j) {
        const int col = at.base(k, j >> 2) + (j & 3);
        return col < a.C ? col : 0;
      };
      float w[kChunkCols], b[kChunkCols];
      with_param(a.w, a.param_dtype, 1.f, [&](auto load) {
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) w[j] = load(column(j));
      });
      with_param(a.b, a.param_dtype, 0.f, [&](auto load) {
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) b[j] = load(column(j));
      });
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[j] = fmaf((v[j] - mean) * rs, w[j], b[j]);
      at.template store<DTY, kVec>(v, a.y + (int64_t)r * a.C * kYB, k);
    }
    if (a.statistics != nullptr && threadIdx.x == 0) a.statistics[r] = make_float2(mean, rs);
  }
}

template <int DTX, int DTY, bool kVec>
__global__ __launch_bounds__(kWideLanes) void norm_wide_bwd_kernel(const NormArgs a) {
  constexpr int kP = norm_pieces<DTX, DTY>(), kXB = ChunkElt<DTX>::kBytes, kYB = ChunkElt<DTY>::kBytes;
  __shared__ typename RowSum<kWideLanes>::Shared s_red;
  RowSum<kWideLanes> sum(&s_red);
  const RowLanes<kWideLanes, 1, kP> at = {(int)threadIdx.x, a.C};
  const int chunks = (a.C + kWideLanes * kChunkCols - 1) / (kWideLanes * kChunkCols);
  for (uint32_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const uint8_t *row = a.row(r), *dy = a.dy + (int64_t)r * a.C * kYB;
    const float2 st = a.statistics[r];
    float v[kChunkCols], g[kChunkCols], s0 = 0.f, s1 = 0.f;
    auto chunk = [&](int k) {  // xh in v, dy w in g; zeros in absent columns of g
      at.template values<DTX, kVec>(at.template load<DTX, kVec, false>(row, k), k, true, false, v);
      at.template values<DTY, kVec>(at.template load<DTY, kVec, false>(dy, k), k, true, false, g);
      float w[kChunkCols];
      with_param(a.w, a.param_dtype, 1.f, [&](auto load) {
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const int col = at.base(k, j >> 2) + (j & 3);
          w[j] = load(col < a.C ? col : 0);
        }
      });
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        v[j] = (v[j] - st.x) * st.y;
        g[j] *= w[j];
      }
    };
    for (int k = 0; k < chunks; ++k) {
      chunk(k);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        s0 += g[j];
        s1 = fmaf(g[j], v[j], s1);
      }
    }
    sum.two(s0, s1);
    s0 = a.layer ? s0 * a.inv_c : 0.f;
    s1 *= a.inv_c;
    for (int k = 0; k < chunks; ++k) {
      chunk(k);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[j] = st.y * (g[j] - s0 - v[j] * s1);
      at.template store<DTX, kVec>(v, a.dx + (int64_t)r * a.C * kXB, k);
    }
  }
}

// The sums over rows where rows are not held: a thread owns eight columns, a
// workgroup 64 threads by 4 rows, slab by slab of rows.
constexpr int kSumLanes = 64, kSumRows = 4;

template <int DTX, int DTY, bool kVec>
__global__ __launch_bounds__(kSumLanes* kSumRows) void norm_columns_kernel(const NormArgs a) {
  constexpr int kP = norm_pieces<DTX, DTY>(), kYB = ChunkElt<DTY>::kBytes;
  __shared__ float s_sum[kSumRows][2][kSumLanes * kChunkCols];
  const int lane = threadIdx.x % kSumLanes, group = threadIdx.x / kSumLanes;
  const RowLanes<kSumLanes, 1, kP> at = {lane, a.C};
  const int k = blockIdx.y;
  float dw[kChunkCols] = {}, db[kChunkCols] = {};
  for (uint32_t r = blockIdx.x * kSumRows + group; r < a.rows; r += gridDim.x * kSumRows) {
    const float2 st = a.statistics[r];
    float v[kChunkCols], g[kChunkCols];
    at.template values<DTX, kVec>(at.template load<DTX, kVec, false>(a.row(r), k), k, true, false, v);
    at.template values<DTY, kVec>(at.template load<DTY, kVec, false>(a.dy + (int64_t)r * a.C * kYB, k), k, true, false, g);
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) {
      dw[j] = fmaf(g[j], (v[j] - st.x) * st.y, dw[j]);
      db[j] += g[j];
    }
  }
#pragma unroll
  for (int j = 0; j < kChunkCols; ++j) {
    const int c = at.base(0, j >> 2) + (j & 3);
    s_sum[group][0][c] = dw[j];
    s_sum[group][1][c] = db[j];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * kSumLanes * kChunkCols; i += kSumLanes * kSumRows) {
    const int which = i / (kSumLanes * kChunkCols), c = i % (kSumLanes * kChunkCols);
    const int64_t col = (int64_t)k * kSumLanes * kChunkCols + c;
    if (col < a.C)
      a.partial[((int64_t)blockIdx.x * 2 + which) * a.C + col] =
          (s_sum[0][which][c] + s_sum[1][which][c]) + (s_sum[2][which][c] + s_sum[3][which][c]);
  }
}

// Row groups of a workgroup of the forward: few, so that workgroups that load and
// such that compute are side by side, but enough for the parameters, 8 C bytes a workgroup,
// to be a small part of what it reads.
template <int DTX, int DTY, int kG, int kK, bool kVec, bool kPairs>
void launch_norm(const NormArgs& a, hipStream_t s) {
  constexpr uint32_t kGroups = tail_threads(kG) / kG, kMostTurns = kG > 64 ? 16 : (kG > 16 ? 4 : 2);
  const uint32_t need = (a.rows + kGroups - 1) / kGroups, few = need >= 512 ? need / 512 : 1;
  const uint32_t turns = few < kMostTurns ? few : kMostTurns, blocks = (need + turns - 1) / turns;
  constexpr uint32_t kMost = 1u << 22;  // a grid holds fewer than 2^32 threads
  norm_kernel<DTX, DTY, kG, kK, kVec, kPairs><<<blocks < kMost ? blocks : kMost, tail_threads(kG), 0, s>>>(a);
}

template <int DTX, int DTY, int kG, int kK, bool kVec, bool kPairs>
void launch_norm_bwd(const NormArgs& a, hipStream_t s) {
  norm_bwd_kernel<DTX, DTY, kG, kK, kVec, kPairs><<<a.parts, tail_threads(kG), 0, s>>>(a);
}

// Workgroups that the compute units hold at once, no more: each reads the parameters of its columns one by one first.
template <int DTX, int DTY, int kG, int kK>
void launch_norm_flat(const NormArgs& a, hipStream_t s) {
  constexpr int kThreads = tail_threads(kG);
  constexpr uint32_t kGroups = kThreads / kG;
  static const uint32_t most = [] {
    int n = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, norm_flat_kernel<DTX, DTY, kG, kK>, kThreads, 0) != hipSuccess || n < 1) {
      (void)hipGetLastError();
      n = 2;
    }
    return 256u * (uint32_t)n;
  }();
  const uint32_t need = ((a.rows + kGroups - 1) / kGroups + 7) / 8 * 8;
  norm_flat_kernel<DTX, DTY, kG, kK><<<need < most ? need : most, kThreads, 0, s>>>(a);
}

template <int DTX, int DTY, int kG, int kK>
void launch_norm_flat_bwd(const NormArgs& a, hipStream_t s) {
  norm_flat_bwd_kernel<DTX, DTY, kG, kK><<<a.parts, tail_threads(kG), 0, s>>>(a);
}

#define TERRA_NORM_FLAT_SHAPES(f, shape, ...)                                                \
  switch ((shape).lanes * 10 + (shape).chunks) {                                             \
    case 81: return f<DTX, DTY, 8, 1>(__VA_ARGS__);                                          \
    case 83: return f<DTX, DTY, 8, 3>(__VA_ARGS__);                                          \
    case 161: return f<DTX, DTY, 16, 1>(__VA_ARGS__);                                        \
    case 162: return f<DTX, DTY, 16, 2>(__VA_ARGS__);                                        \
    case 163: return f<DTX, DTY, 16, 3>(__VA_ARGS__);                                        \
    case 322: return f<DTX, DTY, 32, 2>(__VA_ARGS__);                                        \
    case 323: return f<DTX, DTY, 32, 3>(__VA_ARGS__);                                        \
    case 642: return f<DTX, DTY, 64, 2>(__VA_ARGS__);                                        \
    case 643: return f<DTX, DTY, 64, 3>(__VA_ARGS__);                                        \
    case 644: return f<DTX, DTY, 64, 4>(__VA_ARGS__);                                        \
    case 2562: return f<DTX, DTY, 256, 2>(__VA_ARGS__);                                      \
    case 5122: return f<DTX, DTY, 512, 2>(__VA_ARGS__);                                      \
    default: return f<DTX, DTY, 1024, 2>(__VA_ARGS__);                                       \
  }

template <int DTX, int DTY>
void flat_fwd(const NormArgs& a, const NormPlan& p, hipStream_t s) {
  TERRA_NORM_FLAT_SHAPES(launch_norm_flat, p.shape, a, s)
}

template <int DTX, int DTY>
void flat_bwd(const NormArgs& a, const NormPlan& p, hipStream_t s) {
  TERRA_NORM_FLAT_SHAPES(launch_norm_flat_bwd, p.shape, a, s)
}

#define TERRA_NORM_ROWS(f, g, k, ...)                                                        \
  {                                                                                          \
    if (vec) return f<DTX, DTY, g, k, true, false>(__VA_ARGS__);                             \
    if constexpr (DTX != TERRA_DTYPE_F32 && DTY != TERRA_DTYPE_F32)                          \
      if (pairs) return f<DTX, DTY, g, k, false, true>(__VA_ARGS__);                         \
    return f<DTX, DTY, g, k, false, false>(__VA_ARGS__);                                     \
  }
// Calls f<DTX, DTY, lanes, chunks, kVec, kPairs>(...) for the shape of the call; wide: that of 2049 to 4096 channels.
// 83 is no shape of fp32 pieces, which layer_norm.hip asserts of all widths.
#define TERRA_NORM_SHAPES(f, shape, wide, ...)                                                   \
  switch ((shape).lanes * 10 + (shape).chunks) {                                             \
    case 21: TERRA_NORM_ROWS(f, 2, 1, __VA_ARGS__)                                           \
    case 41: TERRA_NORM_ROWS(f, 4, 1, __VA_ARGS__)                                           \
    case 81: TERRA_NORM_ROWS(f, 8, 1, __VA_ARGS__)                                           \
    case 83: if constexpr (norm_pieces<DTX, DTY>() == 8) TERRA_NORM_ROWS(f, 8, 3, __VA_ARGS__) \
    case 161: TERRA_NORM_ROWS(f, 16, 1, __VA_ARGS__)                                         \
    case 162: TERRA_NORM_ROWS(f, 16, 2, __VA_ARGS__)                                         \
    case 163: TERRA_NORM_ROWS(f, 16, 3, __VA_ARGS__)                                         \
    case 322: TERRA_NORM_ROWS(f, 32, 2, __VA_ARGS__)                                         \
    case 323: TERRA_NORM_ROWS(f, 32, 3, __VA_ARGS__)                                         \
    case 642: TERRA_NORM_ROWS(f, 64, 2, __VA_ARGS__)                                         \
    case 644: TERRA_NORM_ROWS(f, 64, 4, __VA_ARGS__)                                         \
    case wide: TERRA_NORM_ROWS(f, wide / 10, wide % 10, __VA_ARGS__)                         \
    case 5122: TERRA_NORM_ROWS(f, 512, 2, __VA_ARGS__)                                       \
    default: TERRA_NORM_ROWS(f, 1024, 2, __VA_ARGS__)                                        \
  }

template <int DTX, int DTY>
void held_fwd(const NormArgs& a, const NormPlan& p, bool vec, bool pairs, hipStream_t s) {
  TERRA_NORM_SHAPES(launch_norm, p.shape, 648, a, s)
}

template <int DTX, int DTY>
void held_bwd(const NormArgs& a, const NormPlan& p, bool vec, bool pairs, hipStream_t s) {
  TERRA_NORM_SHAPES(launch_norm_bwd, p.shape, 2562, a, s)
}

template <int DTX, int DTY>
void norm_fwd(const NormArgs& a, const NormPlan& p, bool vec, bool pairs, hipStream_t s) {
  if (p.flat) return flat_fwd<DTX, DTY>(a, p, s);
  if (p.held) return held_fwd<DTX, DTY>(a, p, vec, pairs, s);
  const uint32_t blocks = a.rows < (1u << 22) ? a.rows : 1u << 22;  // a grid holds fewer than 2^32 threads
  if (vec) norm_wide_kernel<DTX, DTY, true><<<blocks, kWideLanes, 0, s>>>(a);
  else norm_wide_kernel<DTX, DTY, false><<<blocks, kWideLanes, 0, s>>>(a);
}

template <int DTX, int DTY>
void norm_bwd(const NormArgs& a, const NormPlan& p, bool vec, bool pairs, hipStream_t s) {
  if (p.flat) return flat_bwd<DTX, DTY>(a, p, s);
  if (p.held) return held_bwd<DTX, DTY>(a, p, vec, pairs, s);
  const uint32_t blocks = a.rows < (1u << 22) ? a.rows : 1u << 22;
  if (a.dx != nullptr) {
    if (vec) norm_wide_bwd_kernel<DTX, DTY, true><<<blocks, kWideLanes, 0, s>>>(a);
    else norm_wide_bwd_kernel<DTX, DTY, false><<<blocks, kWideLanes, 0, s>>>(a);
  }
  if (a.partial != nullptr) {
    const dim3 grid(a.parts, (a.C + kSumLanes * kChunkCols - 1) / (kSumLanes * kChunkCols));
    if (vec) norm_columns_kernel<DTX, DTY, true><<<grid, kSumLanes * kSumRows, 0, s>>>(a);
    else norm_columns_kernel<DTX, DTY, false><<<grid, kSumLanes * kSumRows, 0, s>>>(a);
  }
}

}  // namespace
}  // namespace terra

#define TERRA_NORM_DEFINE(x, X, y, Y)                                                                              \
  namespace terra {                                                                                                \
  void norm_fwd_##x##_##y(const void* args, const NormPlan& plan, bool vec, bool pairs, hipStream_t s) {          \
    norm_fwd<TERRA_DTYPE_##X, TERRA_DTYPE_##Y>(*static_cast<const NormArgs*>(args), plan, vec, pairs, s);         \
  }                                                                                                                \
  void norm_bwd_##x##_##y(const void* args, const NormPlan& plan, bool vec, bool pairs, hipStream_t s) {          \
    norm_bwd<TERRA_DTYPE_##X, TERRA_DTYPE_##Y>(*static_cast<const NormArgs*>(args), plan, vec, pairs, s);         \
  }                                                                                                                \
  }
