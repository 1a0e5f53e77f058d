// The end of a half-block, row by row of C channels (residual_norm.hip holds
// the forward, residual_norm_bwd.hip the backward):
//
//   n = post_norm(h)          LayerNorm, RMS norm or nothing, with affine
//   m = keep s n              dropout (row_chunk.h)
//   y = alpha x + gate m      gate [C], one for each sample [B, C], or 1
//   z = next_norm(y)          the norm that the next half-block begins with, or nothing
//
//   LayerNorm(v) = (v - mean v) r w + b,  r = rsqrt(mean (v - mean v)^2 + eps)
//   RMS norm(v)  = v r w + b,             r = rsqrt(mean v^2 + eps)
//
// All of it in fp32 in registers, two-pass statistics, z from the y that is
// not yet rounded; y and z are rounded once each.  h may be in window order: a
// row's source is then the window token that the reverse of the windows and
// the inverse roll bring to it, and m = 0 where no emitted window holds it.
#pragma once

#include "row_chunk.h"

namespace terra {
namespace {

// Grid token -> row of the window tensor, or -1.
struct WindowMap {
  int32_t Hp, Wp, shift_h, shift_w, pad_top, pad_left;
  int32_t row_begin, rows, cols, ws;
  int32_t valid_begin, valid_end;  // valid_end <= 0: all valid
  FastDiv fd_W, fd_H, fd_ws;

  __device__ __forceinline__ int64_t source(uint32_t token) const {
    uint32_t rest, sw, b, sh, wr, ti, wc, tj;
    fd_W.divmod(token, rest, sw);
    fd_H.divmod(rest, b, sh);
    int fi = (int)sh + pad_top - shift_h;
    int fj = (int)sw + pad_left - shift_w;
    if (fi < 0) fi += Hp;
    if (fj < 0) fj += Wp;
    fd_ws.divmod((uint32_t)fi, wr, ti);
    fd_ws.divmod((uint32_t)fj, wc, tj);
    const int wr_l = (int)wr - row_begin;
    const int wl = wr_l * cols + (int)wc;
    const bool have = (unsigned)wr_l < (unsigned)rows && (valid_end <= 0 || (wl >= valid_begin && wl < valid_end));
    const int64_t w = (int64_t)b * rows * cols + wl;
    return have ? w * ws * ws + (int64_t)(ti * ws + tj) : -1;
  }
};

struct TailArgs {
  const uint8_t *h, *x, *dy, *dz;   // dy, dz: backward, either may be NULL (zero)
  uint8_t *y, *z, *dh, *dx;
  const float *pw, *pb, *gate, *nw, *nb;  // NULL: 1 (weights, gate) or 0 (biases)
  float* partial;       // backward: [gridDim.x][4][C], the workgroups' sums for pw, pb, nw, nb
  float* gate_partial;  // backward: [units][C]
  DropoutArgs drop;
  uint32_t rows, per_sample;        // per_sample: rows that share a row of the gate
  int64_t h_row_bytes, x_row_bytes; // of h and x; the other tensors' rows are packed
  int32_t C, post, next;            // post, next: enum terra_norm
  float post_eps, next_eps, alpha, inv_c;
  int32_t gate_rows;                // 0: none, 1: one for all, B: one for each sample
  int32_t windows;                  // h is in window order
  uint32_t slabs, slab_rows, units; // backward: see there
  WindowMap map;
};

// How the lanes hold a row: kG lanes with kK chunks each.
struct TailShape {
  int32_t lanes, chunks;  // per row, per lane
};

// Fewest lanes that hold the row with one chunk each up to a wave; then two
// chunks a lane, then a workgroup for each row.
inline TailShape tail_shape(int C) {
  const int n = (C + kChunkCols - 1) / kChunkCols;
  if (n <= 16) return {16, 1};
  if (n <= 32) return {32, 1};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return {256, 1};
  if (n <= 512) return {256, 2};
  return {512, 2};
}
constexpr int kTailMaxChannels = 8192;

constexpr int tail_threads(int lanes) { return lanes > 256 ? lanes : 256; }

// The statistics of a normalised row held as kK chunks a lane: v becomes
// (v - mean) r (zero in absent columns), r is returned.
template <int kG, int kK, bool kVec>
__device__ __forceinline__ float normalise(float (&v)[kK][kChunkCols], int kind, float eps, float inv_c, int lane, int C,
                                           RowSum<kG>& sum) {
  if (kind == TERRA_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) s += v[k][j];
    const float mean = sum.one(s) * inv_c;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      const int col = (lane + kG * k) * kChunkCols;
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[k][j] = col + (kVec ? 0 : j) < C ? v[k][j] - mean : 0.f;
    }
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < kK; ++k)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) q = fmaf(v[k][j], v[k][j], q);
  const float r = rsqrtf(sum.one(q) * inv_c + eps);
#pragma unroll
  for (int k = 0; k < kK; ++k)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) v[k][j] *= r;
  return r;
}

// Eight parameters of a chunk in fp32, `none` where the pointer is NULL and 0
// in absent columns.
template <bool kVec>
__device__ __forceinline__ void load_params(const float* p, float none, int col, int C, float (&f)[kChunkCols]) {
#pragma unroll
  for (int j = 0; j < kChunkCols; ++j) f[j] = col + (kVec ? 0 : j) < C ? none : 0.f;
  if (p == nullptr) return;
  if constexpr (kVec) {
    if (col < C) {
      const float4 a = *reinterpret_cast<const float4*>(p + col), b = *reinterpret_cast<const float4*>(p + col + 4);
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j)
      if (col + j < C) f[j] = p[col + j];
  }
}

}  // namespace

// The backward's launch, by the types of h and x (residual_norm_bwd.hip).
struct TailBwdPlan {
  TailShape shape;
  uint32_t slabs, slab_rows, units, blocks;
};
TailBwdPlan tail_bwd_plan(uint32_t rows, int C, int gate_rows);
int launch_tail_bwd(int h_dtype, int x_dtype, const void* args, const TailBwdPlan& plan, bool vec, hipStream_t s);

}  // namespace terra
