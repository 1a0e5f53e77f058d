// LayerNorm and RMS norm over rows of C channels, forward and backward:
//
//   xh = (x - mean x) r,  r = rsqrt(mean (x - mean x)^2 + eps)     LayerNorm
//   xh = x r,             r = rsqrt(mean x^2 + eps)                RMS norm
//   y  = xh w + b
//   g  = dy w,  dx = r (g - mean g - xh mean(g xh))   (an RMS norm has no mean g)
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// All of it in fp32, two-pass statistics, y and dx rounded once; the parameters
// are read in their own type and their gradients written in it.  Row r of x begins (r / inner) outer + (r % inner) step
// elements into x, so the heads of a packed q|k|v are rows too; y, dy and dx are packed.
//
// Bound by memory: a row is read once and held in registers through its two sums, in the forward with the next one on
// its way meanwhile (39168 x 4096 bf16: forward 118 us, 5.4 TB/s, backward 161 us, 6.0; 524288 x 192 fp32 to bf16: 94 and
// 167 us; a large copy moves 5.35).  One row of 1024 is a launch (3 us).
// Rows above 16384 channels are read again for each sum by a workgroup a row: 3662 x 16384 bf16 51 and 93 us,
// 1831 x 32768 253 and 294 (1.0 and 1.2 TB/s).
//
// Sums over rows: workgroups keep the sums of the rows that they take in fp32 and write
// them to a workspace, a second launch adds those up in fp64 and rounds once: no atomics, an
// order that the sizes and alignments fix.  (fp64 from the first row on would
// double the registers of the sums.)
#pragma once

#include "residual_norm.h"

namespace terra {
namespace {

struct NormArgs {
  const uint8_t *x, *dy;
  uint8_t *y, *dx;         // dx may be NULL: only sums are asked for
  const void *w, *b;       // NULL: 1, 0
  float2* statistics;      // mean and r of each row, or NULL (forward)
  float* partial;          // backward: [parts][2][C], or NULL: no sums
  uint32_t rows, parts;
  FastDiv inner;
  int64_t outer_bytes, step_bytes;
  int32_t C, param_dtype;
  bool layer;
  float eps, inv_c;

  __device__ __forceinline__ const uint8_t* row(uint32_t r) const {
    uint32_t q, rest;
    inner.divmod(r, q, rest);
    return x + (int64_t)q * outer_bytes + (int64_t)rest * step_bytes;
  }
};

// Calls f(load), where load(c) is parameter c in fp32 (`none` where the pointer is NULL): the type is asked once, so that
// the loads of f stand side by side.
template <typename F>
__device__ __forceinline__ void with_param(const void* p, int dtype, float none, F f) {
  if (p == nullptr) f([&](int) { return none; });
  else if (dtype == TERRA_DTYPE_F32) f([&](int c) { return reinterpret_cast<const float*>(p)[c]; });
  else if (dtype == TERRA_DTYPE_BF16) f([&](int c) { return bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[c]); });
  else f([&](int c) { return __half2float(__ushort_as_half(reinterpret_cast<const uint16_t*>(p)[c])); });
}

// A parameter of a row's lanes: in LDS where rows share a workgroup (kG <= 64; the caller adds the
// barrier), else, each lane's columns being its own, in registers.  0 in absent columns.
template <int kG, int kK, int kP>
struct NormParam {
  static constexpr bool kLds = kG <= 64;
  static constexpr int kCols = kG * kK * kChunkCols, kThreads = tail_threads(kG);
  struct Shared { __attribute__((aligned(16))) float v[kLds ? kCols : 4]; };
  Shared* s;
  float r[kLds ? 1 : kK][kChunkCols];

  __device__ __forceinline__ explicit NormParam(Shared* shared) : s(shared) {}

  template <bool kVec>
  __device__ __forceinline__ void fill(const RowLanes<kG, kK, kP>& at, const void* p, int dtype, float none) {
    const int C = at.C;
    with_param(p, dtype, none, [&](auto load) {
      if constexpr (kLds) {
        for (int c = threadIdx.x; c < kCols; c += kThreads) s->v[c] = c < C ? load(c) : 0.f;
      } else {
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = at.base(k, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // kVec: four at once
              const bool has = at.template has<kVec>(k, 4 * h + j);
              const float v = load(kVec ? (has ? col : 0) + j : (has ? col + j : 0));
              r[k][4 * h + j] = has ? v : 0.f;
            }
          }
      }
    });
  }
  __device__ __forceinline__ void get(int k, const RowLanes<kG, kK, kP>& at, float (&f)[kChunkCols]) const {
    if constexpr (kLds) {
      const float4 lo = *reinterpret_cast<const float4*>(&s->v[at.base(k, 0)]);
      const float4 hi = *reinterpret_cast<const float4*>(&s->v[at.base(k, 1)]);
      f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
    } else {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) f[j] = r[k][j];
    }
  }
};

// The statistics of a row held as kK chunks a lane: v becomes xh (zero in
// absent columns), r is returned.
template <int kG, int kK, int kP, bool kVec>
__device__ __forceinline__ float norm_row(float (&v)[kK][kChunkCols], bool layer, float eps, float inv_c,
                                          const RowLanes<kG, kK, kP>& at, RowSum<kG>& sum, float& mean) {
  mean = 0.f;
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) s += v[k][j];
    mean = sum.one(s) * inv_c;
  }
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < kK; ++k)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) {
      v[k][j] -= at.template has<kVec>(k, j) ? mean : 0.f;  // kVec: one select for four
      q = fmaf(v[k][j], v[k][j], q);
    }
  const float r = rsqrtf(sum.one(q) * inv_c + eps);
#pragma unroll
  for (int k = 0; k < kK; ++k)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) v[k][j] *= r;
  return r;
}

}  // namespace

// The kernels' launches by the types of x and y, each with a source file of
// its own; `args` is a NormArgs.
struct NormPlan {
  uint32_t parts;  // workgroups of the sums over rows
  bool held;       // rows are held in registers (else read again)
  bool flat;       // and read by the aligned chunks of the packed tensor
  TailShape shape;
};
#define TERRA_NORM_TYPES(X) X(f32, f32) X(f32, bf16) X(f32, f16) X(bf16, bf16) X(bf16, f32) X(f16, f16) X(f16, f32)
#define TERRA_NORM_DECLARE(x, y)                                                        \
  void norm_fwd_##x##_##y(const void* args, const NormPlan& plan, bool vec, bool pairs, hipStream_t s); \
  void norm_bwd_##x##_##y(const void* args, const NormPlan& plan, bool vec, bool pairs, hipStream_t s);
TERRA_NORM_TYPES(TERRA_NORM_DECLARE)

}  // namespace terra
