// The end of a half-block, row by row of C channels (residual_norm_fwd.h and
// residual_norm_bwd.h hold the kernels, residual_norm.hip the entry points):
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

// What a launch has.  The first three are template parameters of the kernels:
// tested at run time they cost the rows' loops a register copy of every value
// that either side of a test may hold, and the backward of three chunks a lane the
// room for a second wave (524288 x 192 bf16: 276 us, 253 so).
enum TailFlags : uint32_t {
  kTailPost = 1,       // a post-norm
  kTailNext = 2,       // a next norm (backward: whose gradient is given)
  kTailDrop = 4,
  kTailFeatures = 7,
  kTailAtRunTime = 8,  // as a template parameter: the first three are the call's flags
  kTailPostLayer = 16, kTailNextLayer = 32,  // the norm is a LayerNorm
  kTailWindows = 64,   // h is in window order
  kTailDy = 128,       // backward: the gradient of y is given
  kTailPairs = 256,    // rows that are not of whole aligned chunks begin at, and hold, whole aligned pairs of 16-bit columns
};

struct TailArgs {
  const uint8_t *h, *x, *dy, *dz;   // dy, dz: backward, either may be NULL (zero)
  uint8_t *y, *z, *dh, *dx;
  const float *pw, *pb, *gate, *nw, *nb;  // NULL: 1 (weights, gate) or 0 (biases)
  float* partial;       // backward: [gridDim.x][4][C], the workgroups' sums for pw, pb, nw, nb
  float* gate_partial;  // backward: [units][C]
  int32_t branch_sums;  // backward: pw's, pb's or the gate's gradient is asked for
  DropoutArgs drop;
  uint32_t rows, per_sample;        // per_sample: rows that share a row of the gate
  int64_t h_row_bytes, x_row_bytes; // of h and x; the other tensors' rows are packed
  int32_t C;
  uint32_t flags;                   // TailFlags
  float post_eps, next_eps, alpha, inv_c;
  int32_t gate_rows;                // 0: none, 1: one for all, B: one for each sample
  uint32_t slabs, units;            // backward: see there
  WindowMap map;
};

template <int kF>
__device__ __forceinline__ bool tail_has(const TailArgs& a, uint32_t feature) {
  return ((uint32_t)kF & kTailAtRunTime ? a.flags : (uint32_t)kF) & feature;
}

// How the lanes hold a row: kG lanes with kK chunks each.
struct TailShape {
  int32_t lanes, chunks;  // per row, per lane
};

// Where a lane's values stand: value j of its chunk k is column base(k, j / 4) + j % 4.
// With a 16-bit x the chunk is eight columns in a row (16 bytes a load).  An fp32 x
// is accessed 16 bytes, four columns, a lane, neighbouring lanes side by
// side, and the chunk is two such pieces kG lanes apart: eight columns in a row would
// be two loads of every other 16 bytes, each line fetched, and worse, written,
// in two halves (524288 x 192, bf16 h and fp32 x, forward: 365 us against 229).
template <int kG, int kK, int kP>
struct RowLanes {
  static_assert(kP == 8 || kP == 4, "columns a lane holds side by side");
  int lane, C;
  __device__ __forceinline__ int base(int k, int half) const {
    return kP == 8 ? (lane + kG * k) * 8 + 4 * half : (lane + kG * (2 * k + half)) * 4;
  }
  template <bool kVec>
  __device__ __forceinline__ bool has(int k, int j) const { return base(k, j >> 2) + (kVec ? 0 : (j & 3)) < C; }

  // The lane's chunk k of the row at `row`, whose addresses are valid; absent columns read column 0.
  // kPairs: as kTailPairs.
  template <int DT, bool kVec, bool kPairs>
  __device__ __forceinline__ RowChunk<DT> load(const uint8_t* row, int k) const {
    constexpr int kB = ChunkElt<DT>::kBytes;
    RowChunk<DT> r;
    if constexpr (kVec && (kB == 4 || kP == 4)) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int col = base(k, q);
        const uint8_t* p = row + (col < C ? (int64_t)col * kB : 0);
        if constexpr (kB == 4) {
          r.q[q] = __builtin_nontemporal_load(reinterpret_cast<const stream_u32x4*>(p));
        } else {
          const stream_u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const stream_u32x2*>(p));
          r.q[0][2 * q] = v[0];
          r.q[0][2 * q + 1] = v[1];
        }
      }
    } else if constexpr (kVec) {
      const int col = base(k, 0);
      r.q[0] = __builtin_nontemporal_load(reinterpret_cast<const stream_u32x4*>(row + (col < C ? (int64_t)col * kB : 0)));
    } else if constexpr (kB == 2 && kPairs) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = base(k, i >> 1) + 2 * (i & 1);
        r.q[0][i] = *reinterpret_cast<const uint32_t*>(row + (at < C ? (int64_t)at * kB : 0));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        const int at = base(k, j >> 2) + (j & 3), c = at < C ? at : 0;
        if constexpr (kB == 4) {
          r.q[j >> 2][j & 3] = reinterpret_cast<const uint32_t*>(row)[c];
        } else {
          const uint32_t v = reinterpret_cast<const uint16_t*>(row)[c];
          r.q[0][j >> 1] = j & 1 ? r.q[0][j >> 1] | (v << 16) : v;
        }
      }
    }
    return r;
  }

  // Its values in fp32, zeros in absent columns and where the row is not there.
  // all: (uniform) no lane of the launch has either, which spares the selects.
  template <int DT, bool kVec>
  __device__ __forceinline__ void values(RowChunk<DT> r, int k, bool there, bool all, float (&f)[kChunkCols]) const {
    if (!kVec || !all) {
#pragma unroll
      for (int i = 0; i < RowChunk<DT>::kWords; ++i)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int j = ChunkElt<DT>::kBytes == 4 ? 4 * i + w : 2 * w;
          uint32_t v = there && has<kVec>(k, j) ? r.q[i][w] : 0u;
          if constexpr (!kVec && ChunkElt<DT>::kBytes == 2) v = has<false>(k, j + 1) ? v : v & 0xffffu;
          r.q[i][w] = v;
        }
    }
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) f[j] = chunk_value<DT>(r, j);
  }

  // Stores chunk k, rounded once, into the row at `row`, which begins `off` bytes into the descriptor's range.
  template <int DT, bool kVec>
  __device__ __forceinline__ void store(const float (&f)[kChunkCols], __amdgpu_buffer_rsrc_t out, uint32_t off, uint8_t* row, int k) const {
    constexpr uint32_t kB = ChunkElt<DT>::kBytes;
    if constexpr (kVec && kB == 2 && kP == 8) {
      const int col = base(k, 0);
      if (col < C)
        stream_store_sc1(stream_u32x4{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]),
                                      pack2<DT>(f[6], f[7])}, out, off + (uint32_t)col * kB);
    } else if constexpr (kVec) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int col = base(k, q);
        if (col >= C) continue;
        if constexpr (kB == 4)
          stream_store_sc1(stream_u32x4{__float_as_uint(f[4 * q]), __float_as_uint(f[4 * q + 1]), __float_as_uint(f[4 * q + 2]),
                                        __float_as_uint(f[4 * q + 3])}, out, off + (uint32_t)col * kB);
        else
          stream_store_sc1(stream_u32x2{pack2<DT>(f[4 * q], f[4 * q + 1]), pack2<DT>(f[4 * q + 2], f[4 * q + 3])}, out,
                           off + (uint32_t)col * kB);
      }
    } else {
      store_half<DT>(f, row, base(k, 0), C);
      store_half<DT>(f + 4, row, base(k, 1), C);
    }
  }

  // The same into the row at `row`, a place of each row's own.
  template <int DT, bool kVec>
  __device__ __forceinline__ void store(const float (&f)[kChunkCols], uint8_t* row, int k) const {
    constexpr int kB = ChunkElt<DT>::kBytes;
    if constexpr (kVec && kB == 2 && kP == 8) {
      const int col = base(k, 0);
      if (col < C)
        __builtin_nontemporal_store(stream_u32x4{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]),
                                                 pack2<DT>(f[6], f[7])},
                                    reinterpret_cast<stream_u32x4*>(row + (int64_t)col * kB));
    } else if constexpr (kVec) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int col = base(k, q);
        if (col >= C) continue;
        if constexpr (kB == 4)
          __builtin_nontemporal_store(stream_u32x4{__float_as_uint(f[4 * q]), __float_as_uint(f[4 * q + 1]),
                                                   __float_as_uint(f[4 * q + 2]), __float_as_uint(f[4 * q + 3])},
                                      reinterpret_cast<stream_u32x4*>(row + (int64_t)col * kB));
        else
          __builtin_nontemporal_store(stream_u32x2{pack2<DT>(f[4 * q], f[4 * q + 1]), pack2<DT>(f[4 * q + 2], f[4 * q + 3])},
                                      reinterpret_cast<stream_u32x2*>(row + (int64_t)col * kB));
      }
    } else {
      store_half<DT>(f, row, base(k, 0), C);
      store_half<DT>(f + 4, row, base(k, 1), C);
    }
  }

  // The draws of chunk k's eight values; without dropout never below the threshold.
  __device__ __forceinline__ ChunkDraws draws(bool drop, uint64_t seed, int k, uint32_t row, uint32_t stream) const {
    if (!drop) return {{~0u, ~0u, ~0u, ~0u}};
    if constexpr (kP == 8) {
      return chunk_draws(seed, (uint32_t)(lane + kG * k), row, stream);
    } else {
      const uint32_t first = (uint32_t)((lane >> 1) + kG * k);
      return half_draws(seed, lane & 1, first, first + kG / 2, row, stream);
    }
  }
};

// Few idle lanes, and the most chunks a lane that leave room for waves to run
// side by side: what a row costs beside its values (addresses, sums over lanes,
// row tests) is paid once for all chunks of a lane.  most: three chunks, but two
// in the backward of an fp32 x, whose registers then hold two waves a SIMD
// (524288 x 192, bf16 h: 347 us, with three 693) or of rows that are not aligned, whose
// single columns take more (524288 x 190 bf16: 530 us, with three 1091).  Eight lanes a row only where
// columns stand eight by eight: as 16-byte pieces of fp32 they would read a
// 16-bit h in runs of 64 bytes.  From 129 chunks on a workgroup holds the row.
constexpr TailShape tail_shape(int C, bool pieces, int most) {
  const int n = (C + kChunkCols - 1) / kChunkCols;
  if (n > 512) return {512, 2};
  if (n > 256) return {512, 1};
  if (n > 128) return {256, 1};
  if (n <= 16) return {16, 1};
  if (n <= 24 && most == 3 && !pieces) return {8, 3};
  if (n <= 32) return {16, 2};
  if (n <= 48 && most == 3) return {16, 3};
  if (n <= 64) return {32, 2};
  if (n <= 96 && most == 3) return {32, 3};
  return {64, 2};
}
inline bool tail_pieces(int x_dtype) { return x_dtype == TERRA_DTYPE_F32; }
inline int tail_bwd_most(int x_dtype, bool vec) { return x_dtype == TERRA_DTYPE_F32 || !vec ? 2 : 3; }
constexpr int kTailMaxChannels = 8192;

constexpr int tail_threads(int lanes) { return lanes > 256 ? lanes : 256; }

// The statistics of a normalised row held as kK chunks a lane: v becomes
// (v - mean) r (zero in absent columns), r is returned.
template <int kG, int kK, int kP, bool kVec>
__device__ __forceinline__ float normalise(float (&v)[kK][kChunkCols], bool layer, float eps, float inv_c,
                                           const RowLanes<kG, kK, kP>& at, RowSum<kG>& sum) {
  float mean = 0.f;
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kK; ++k)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) s += v[k][j];
    mean = sum.one(s) * inv_c;
  }
#pragma unroll
  for (int k = 0; k < kK; ++k)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) v[k][j] -= at.template has<kVec>(k, j) ? mean : 0.f;  // kVec: one select for four
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

// A parameter, `none` where the pointer is NULL.
__device__ __forceinline__ float param_at(const float* p, float none, int c) { return p == nullptr ? none : p[c]; }

// The branch's affine map with the gate and the dropout scale in it:
//   gate * s * (nhat w + b) = nhat gw + gb
__device__ __forceinline__ void branch_params(const TailArgs& a, const float* gate, int c, float& gw, float& gb) {
  const float g = param_at(gate, 1.f, c) * a.drop.scale;
  gw = g * param_at(a.pw, 1.f, c);
  gb = g * param_at(a.pb, 0.f, c);
}

// Per-column parameters of a row's lanes: in LDS where rows share a workgroup
// (kG <= 64), else, each lane's columns being its own, in registers, but for the
// backward of the widest rows, which has none left.
template <int kN, int kG, int kK, int kP>
struct ColumnParams {
  static constexpr bool kLds = kG <= 64 || (kN == 3 && kK > 1);
  static constexpr int kCols = kG * kK * kChunkCols, kThreads = tail_threads(kG);
  struct Shared { __attribute__((aligned(16))) float v[kLds ? kN : 1][kLds ? kCols : 4]; };
  Shared* s;
  float r[kLds ? 1 : kN][kLds ? 1 : kK][kChunkCols];

  __device__ __forceinline__ explicit ColumnParams(Shared* shared) : s(shared) {}

  // f(column, out[kN]) for every column below C; 0 in absent ones.  With LDS the caller adds the barriers.
  template <typename F>
  __device__ __forceinline__ void fill(const RowLanes<kG, kK, kP>& at, F f) {
    const int C = at.C;
    if constexpr (kLds) {
      for (int c = threadIdx.x; c < kCols; c += kThreads) {
        float v[kN] = {};
        if (c < C) f(c, v);
#pragma unroll
        for (int i = 0; i < kN; ++i) s->v[i][c] = v[i];
      }
    } else {
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const int c = at.base(k, j >> 2) + (j & 3);
          float v[kN] = {};
          if (c < C) f(c, v);
#pragma unroll
          for (int i = 0; i < kN; ++i) r[i][k][j] = v[i];
        }
    }
  }
  // At the top of a loop over rows: the parameters are read from LDS in each
  // turn.  The compiler would otherwise hold all of them in registers over the
  // loop, and the waves for which there is then no room are worth more.
  __device__ __forceinline__ void stay() const {
    if constexpr (kLds) asm volatile("" ::: "memory");
  }
  __device__ __forceinline__ void get(int i, int k, const RowLanes<kG, kK, kP>& at, float (&f)[kChunkCols]) const {
    if constexpr (kLds) {
      const float4 lo = *reinterpret_cast<const float4*>(&s->v[i][at.base(k, 0)]);
      const float4 hi = *reinterpret_cast<const float4*>(&s->v[i][at.base(k, 1)]);
      f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
    } else {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) f[j] = r[i][k][j];
    }
  }
};

// Calls f<DTH, DTX, lanes, chunks, kVec, features>(...) for the call's shape and
// features: those of aligned rows each have kernels of their own, other rows one for all,
// or two: 16-bit columns read by pairs where they can be (262144 x 382 bf16: forward
// 256 us, one by one 289, backward 397 and 492; as a run-time choice, 1009 one by one).
#define TERRA_TAIL_FEATURES(f, g, k, features, vec, ...)                                                      \
  if (!(vec)) {                                                                                               \
    if constexpr (DTH != TERRA_DTYPE_F32)                                                                     \
      if ((features) & kTailPairs) return f<DTH, DTX, g, k, false, kTailAtRunTime | kTailPairs>(__VA_ARGS__); \
    return f<DTH, DTX, g, k, false, kTailAtRunTime>(__VA_ARGS__);                                             \
  }                                                                                                           \
  switch ((features) & kTailFeatures) {                                                                       \
    case 0: return f<DTH, DTX, g, k, true, 0>(__VA_ARGS__);                                                   \
    case 1: return f<DTH, DTX, g, k, true, 1>(__VA_ARGS__);                                                   \
    case 2: return f<DTH, DTX, g, k, true, 2>(__VA_ARGS__);                                                   \
    case 3: return f<DTH, DTX, g, k, true, 3>(__VA_ARGS__);                                                   \
    case 4: return f<DTH, DTX, g, k, true, 4>(__VA_ARGS__);                                                   \
    case 5: return f<DTH, DTX, g, k, true, 5>(__VA_ARGS__);                                                   \
    case 6: return f<DTH, DTX, g, k, true, 6>(__VA_ARGS__);                                                   \
    default: return f<DTH, DTX, g, k, true, 7>(__VA_ARGS__);                                                  \
  }
#define TERRA_TAIL_SHAPES(f, shape, most, features, vec, ...)                                                 \
  if constexpr ((most) == 3) {                                                                                \
    if constexpr (DTX != TERRA_DTYPE_F32)                                                                     \
      if ((shape).lanes == 8) { TERRA_TAIL_FEATURES(f, 8, 3, features, vec, __VA_ARGS__) }                    \
    if ((shape).chunks == 3 && (shape).lanes == 16) { TERRA_TAIL_FEATURES(f, 16, 3, features, vec, __VA_ARGS__) } \
    if ((shape).chunks == 3) { TERRA_TAIL_FEATURES(f, 32, 3, features, vec, __VA_ARGS__) }                    \
  }                                                                                                           \
  switch ((shape).lanes * 10 + (shape).chunks) {                                                              \
    case 161: { TERRA_TAIL_FEATURES(f, 16, 1, features, vec, __VA_ARGS__) }                                   \
    case 162: { TERRA_TAIL_FEATURES(f, 16, 2, features, vec, __VA_ARGS__) }                                   \
    case 322: { TERRA_TAIL_FEATURES(f, 32, 2, features, vec, __VA_ARGS__) }                                   \
    case 642: { TERRA_TAIL_FEATURES(f, 64, 2, features, vec, __VA_ARGS__) }                                   \
    case 2561: { TERRA_TAIL_FEATURES(f, 256, 1, features, vec, __VA_ARGS__) }                                 \
    case 5121: { TERRA_TAIL_FEATURES(f, 512, 1, features, vec, __VA_ARGS__) }                                 \
    default: { TERRA_TAIL_FEATURES(f, 512, 2, features, vec, __VA_ARGS__) }                                   \
  }

}  // namespace

// The backward's grid, by the sizes of the call (residual_norm.hip).
struct TailBwdPlan {
  TailShape shape;
  uint32_t slabs, units, blocks;
};

// The kernels' launches by the types of h and x, each with a source file of its
// own; `args` is a TailArgs.
#define TERRA_TAIL_TYPES(X) X(f32, f32) X(bf16, bf16) X(bf16, f32) X(f16, f16) X(f16, f32)
#define TERRA_TAIL_DECLARE(h, x)                                \
  void tail_fwd_##h##_##x(const void* args, bool vec, hipStream_t s); \
  void tail_bwd_##h##_##x(const void* args, const TailBwdPlan& plan, bool vec, hipStream_t s);
TERRA_TAIL_TYPES(TERRA_TAIL_DECLARE)

}  // namespace terra
