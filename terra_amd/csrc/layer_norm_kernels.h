// The kernels of layer_norm.h for one pair of types of x and y.
#pragma once

#include "layer_norm.h"

namespace terra {
namespace {

// ---- rows of any width, read again for each pass --------------------------------
// A workgroup a row; what a pass reads again comes from L2.
constexpr int kWideLanes = 512;

template <int DTX, int DTY>
constexpr int norm_pieces() { return DTX == TERRA_DTYPE_F32 || DTY == TERRA_DTYPE_F32 ? 4 : 8; }

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
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        const int col = at.base(k, j >> 2) + (j & 3), c = col < a.C ? col : 0;
        v[j] = fmaf((v[j] - mean) * rs, norm_param(a.w, a.param_dtype, 1.f, c), norm_param(a.b, a.param_dtype, 0.f, c));
      }
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
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        const int col = at.base(k, j >> 2) + (j & 3);
        v[j] = (v[j] - st.x) * st.y;
        g[j] *= col < a.C ? norm_param(a.w, a.param_dtype, 1.f, col) : 0.f;
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

template <int DTX, int DTY>
void norm_fwd(const NormArgs& a, const NormPlan&, bool vec, bool, hipStream_t s) {
  const uint32_t blocks = a.rows < (1u << 22) ? a.rows : 1u << 22;  // a grid holds fewer than 2^32 threads
  if (vec) norm_wide_kernel<DTX, DTY, true><<<blocks, kWideLanes, 0, s>>>(a);
  else norm_wide_kernel<DTX, DTY, false><<<blocks, kWideLanes, 0, s>>>(a);
}

template <int DTX, int DTY>
void norm_bwd(const NormArgs& a, const NormPlan&, bool vec, bool, hipStream_t s) {
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
