// Dropout whose mask is drawn from a counter-based generator and never stored,
// alone and after the MLP's GELU (between fc1 and fc2), with the backward of
// the latter.  For row r and column c of [rows, C], with keep and s of
// row_chunk.h:
//
//   dropout         y  = keep s x               (its own backward: dx = keep s dy)
//   gelu_dropout    a  = keep s GELU(h),        GELU(h) = h Phi(h) = h erfc(-h / sqrt 2) / 2
//   its backward    dh = keep s da (Phi(h) + h phi(h)),  colsum[c] = sum over r of dh (before its rounding)
//
// A dropped element is 0 whatever its value was.  Each value is computed in
// fp32 and rounded once.
//
// Layout: a thread owns eight columns and steps through rows, so column sums
// stay in its registers; a workgroup is T such threads by R rows.
//
// Bound by memory: 2 values an element moved, 3 in the backward.  524288 x 768:
// dropout bf16 271 us and fp32 (262144 rows) 275, GELU 318, backward 410, with
// column sums 483; a large copy moves the same bytes in 310, 310, 310, 465, 465.
#include "gelu.h"
#include "row_chunk.h"

#include <math.h>

namespace terra {
namespace {

enum DropOp { kDropout = 0, kGeluFwd = 1, kGeluBwd = 2, kGeluBwdSum = 3 };

constexpr int kDropThreads = 256;  // at most, per workgroup
constexpr int kDropRows = 4;       // rows a thread loads before it computes

struct DropParams {
  const uint8_t* in;   // x, h, or da
  const uint8_t* h;    // backward
  uint8_t* out;
  float* partial;      // [gridDim.x][C] column sums
  DropoutArgs drop;
  uint32_t rows;
  int32_t C;
  int64_t row_bytes;     // of out (and of in but for dropout)
  int64_t in_row_bytes;
  int32_t T, R;
};

// Phi(h) and, up to 1 / sqrt(2 pi), phi(h).  With a = |h| and e = exp(-a^2 / 2),
// Phi(-a) = e G(a), where G(a) = erfcx(a / sqrt 2) / 2 falls smoothly from 1/2 like
// 1 / a: a polynomial of degree 8 in u = 1 / (1 + 0.3 a) without a constant term,
// fitted to the least largest relative error over 0 <= a <= 14 (1.5e-7; in fp32
// 2.5e-7 absolute for h > 0).  So the tail does not vanish as 1 + erf does, but its
// relative error grows with the exponent, whose fp32 product is rounded twice: 5.5e-7
// down to h = -2, 1.6e-6 at -5, 3.8e-6 at -9, 7.7e-6 at -12.9, beyond which it is below
// the smallest normal number.  About 20 instructions, of which exp2 and the
// reciprocal go to the transcendental unit; erfcf and expf took three times as many.
__device__ __forceinline__ void normal_parts(float h, float& cdf, float& e) {
  const float a = fabsf(h);
  const float u = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
  e = __builtin_amdgcn_exp2f(-0.72134752044448170f * (h * h));
  float p = 0.0356753467f;
  p = fmaf(p, u, -0.157205686f);
  p = fmaf(p, u, 0.20635832f);
  p = fmaf(p, u, -0.0536883323f);
  p = fmaf(p, u, 0.128564218f);
  p = fmaf(p, u, 0.0999126806f);
  p = fmaf(p, u, 0.120754089f);
  p = fmaf(p, u, 0.11962929f);
  const float q = p * u * e;
  cdf = h > 0.f ? 1.f - q : q;
}

__device__ __forceinline__ float gelu_factor(float h) {
  float cdf, e;
  normal_parts(h, cdf, e);
  return cdf;
}

__device__ __forceinline__ float gelu_slope_of(float h) {
  float cdf, e;
  normal_parts(h, cdf, e);
  return fmaf(0.39894228040143268f * h, e, cdf);
}

// What an element is multiplied by, without the mask: s, s Phi(h), or s times the slope at h.
template <int kOp>
__device__ __forceinline__ float drop_factor(float h, float scale) {
  if constexpr (kOp == kDropout) return scale;
  else if constexpr (kOp == kGeluFwd) return gelu_factor(h) * scale;
  else return gelu_slope_of(h) * scale;
}

// The same by table for a bf16 h: one of 2^16 values, of which those with
// 2^-12 <= |h| < 16 are read from an fp32 table that the workgroup fills with
// drop_factor (gelu.h's layout); beyond 16 the last entries are the limits (1
// and 0, exp(-127) being 0 in fp32), and a wave with a smaller value, an infinity or
// a NaN computes its chunk.  For the forward, which is bound by instructions
// without it (524288 x 768: 318 us against 390); the backward reads a third more and is as fast without (492 against 495).
template <int kOp>
__device__ __forceinline__ void table_factors(const stream_u32x4& h, const uint8_t* table, float scale, float (&f)[kChunkCols]) {
  u16x2 dmax = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) slope_pair(h[i], table, dmax, f[2 * i], f[2 * i + 1]);
  const uint32_t dm = dmax.x > dmax.y ? dmax.x : dmax.y;
  if (__builtin_amdgcn_ballot_w64(dm >= kSlopeRare) != 0)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j)
      f[j] = drop_factor<kOp>(__uint_as_float(j & 1 ? h[j >> 1] & 0xffff0000u : h[j >> 1] << 16), scale);
}

// kPairs: rows that are not of whole aligned chunks, but begin at and hold whole aligned pairs of 16-bit columns.
template <int kOp, int DT, bool kVec, bool kTable, bool kPairs>
__global__ __launch_bounds__(kDropThreads) void drop_kernel(const DropParams a) {
  constexpr int kB = ChunkElt<DT>::kBytes;
  constexpr bool kBwd = kOp >= kGeluBwd;
  constexpr bool kSum = kOp == kGeluBwdSum;
  __shared__ float s_sum[kSum ? kDropThreads * kChunkCols : 1];
  static_assert(!kTable || (kVec && DT == TERRA_DTYPE_BF16 && kOp == kGeluFwd), "the table is of bf16 values");
  __shared__ __attribute__((aligned(16))) float s_table[kTable ? 2 * kSlopeTabSpan : 4];
  if constexpr (kTable) {
    for (int e = threadIdx.x; e < 2 * kSlopeTabSpan; e += blockDim.x) {
      const uint32_t bits = e < kSlopeTabSpan ? kSlopeTabLo + e : 0x8000u + kSlopeTabLo + (e - kSlopeTabSpan);
      s_table[e] = drop_factor<kOp>(__uint_as_float(bits << 16), a.drop.scale);
    }
    __syncthreads();
  }
  const int tc = threadIdx.x % a.T, tr = threadIdx.x / a.T;
  const int strip_col = blockIdx.y * a.T * kChunkCols;
  const int64_t strip = (int64_t)strip_col * kB;  // bytes before this strip of columns
  // The thread's columns: c[0] .. c[0] + 3 and c[1] .. c[1] + 3 of the strip (see row_chunk.h).
  const int c[2] = {kB == 2 ? tc * 8 : tc * 4, kB == 2 ? tc * 8 + 4 : (tc + a.T) * 4};
  const int width = a.C - strip_col;  // columns from the strip's first one on
  const bool present = tr < a.R && c[0] < width;
  auto load = [&](const uint8_t* row) {
    RowChunk<DT> r;
    if constexpr (kVec) {
#pragma unroll
      for (int q = 0; q < RowChunk<DT>::kWords; ++q)
        r.q[q] = __builtin_nontemporal_load(
            reinterpret_cast<const stream_u32x4*>(row + (present && c[q] < width ? strip + c[q] * kB : 0)));
    } else if constexpr (kPairs) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = c[i >> 1] + 2 * (i & 1);
        r.q[0][i] = *reinterpret_cast<const uint32_t*>(row + (present && at < width ? strip + (int64_t)at * kB : 0));
      }
    } else {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        const int at = c[j >> 2] + (j & 3);
        const int64_t col = present && at < width ? strip_col + at : 0;
        if constexpr (kB == 4) {
          r.q[j >> 2][j & 3] = reinterpret_cast<const uint32_t*>(row)[col];
        } else {
          const uint32_t v = reinterpret_cast<const uint16_t*>(row)[col];
          r.q[0][j >> 1] = j & 1 ? r.q[0][j >> 1] | (v << 16) : v;
        }
      }
    }
    return r;
  };
  const uint64_t seed = a.drop.threshold > 0 ? *a.drop.seed : 0;
  float acc[kSum ? kChunkCols : 1];
  if constexpr (kSum)
#pragma unroll
    for (int j = 0; j < kChunkCols; ++j) acc[j] = 0.f;

  const uint64_t step = (uint64_t)gridDim.x * a.R * kDropRows;
  for (uint64_t r0 = (uint64_t)blockIdx.x * a.R * kDropRows; r0 < a.rows; r0 += step) {
    RowChunk<DT> v[kDropRows], hv[kDropRows];
#pragma unroll
    for (int i = 0; i < kDropRows; ++i) {
      const uint64_t row = r0 + (uint64_t)(i * a.R + tr);
      const int64_t r = row < a.rows ? (int64_t)row : (int64_t)a.rows - 1;  // a row past the end re-reads the last one
      v[i] = load(a.in + r * a.in_row_bytes);
      if constexpr (kBwd) hv[i] = load(a.h + r * a.row_bytes);
    }
#pragma unroll
    for (int i = 0; i < kDropRows; ++i) {
      const uint64_t base = r0 + (uint64_t)(i * a.R);
      if (base >= a.rows) break;  // uniform
      const uint32_t live = (uint32_t)(a.rows - base < (uint64_t)a.R ? a.rows - base : (uint64_t)a.R);
      // From this strip's first column of the step's first row on; its bytes end with the step's last row.
      const int64_t left = (int64_t)live * a.row_bytes - strip;
      const __amdgpu_buffer_rsrc_t out =
          buffer_rsrc(a.out + (int64_t)base * a.row_bytes + strip, (uint32_t)(left < 0x7fffffff ? left : 0x7fffffff));
      if (!present || (uint32_t)tr >= live) continue;
      float f[kChunkCols], w[kChunkCols];
      const RowChunk<DT>& at = kBwd ? hv[i] : v[i];  // where the factor is taken
      if constexpr (kTable) {
        table_factors<kOp>(at.q[0], reinterpret_cast<const uint8_t*>(s_table), a.drop.scale, w);
      } else {
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) w[j] = drop_factor<kOp>(chunk_value<DT>(at, j), a.drop.scale);
      }
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) f[j] = chunk_value<DT>(v[i], j) * w[j];
      if (a.drop.threshold > 0) {
        const uint32_t row = (uint32_t)base + (uint32_t)tr, first = (uint32_t)((strip_col + c[0]) / kChunkCols);
        const ChunkDraws d = kB == 2 ? chunk_draws(seed, first, row, a.drop.stream)
                                     : half_draws(seed, tc & 1, first, first + a.T / 2, row, a.drop.stream);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) f[j] = kept(d, j, a.drop.threshold) ? f[j] : 0.f;
      }
      if constexpr (kSum)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) acc[j] += f[j];
      const uint32_t off = (uint32_t)((int64_t)tr * a.row_bytes);
      if constexpr (kVec && kB == 2) {
        stream_store_sc1(stream_u32x4{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3]), pack2<DT>(f[4], f[5]),
                                      pack2<DT>(f[6], f[7])}, out, off + (uint32_t)(c[0] * kB));
      } else if constexpr (kVec) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          if (c[q] < width)
            stream_store_sc1(stream_u32x4{__float_as_uint(f[4 * q]), __float_as_uint(f[4 * q + 1]),
                                          __float_as_uint(f[4 * q + 2]), __float_as_uint(f[4 * q + 3])}, out,
                             off + (uint32_t)(c[q] * kB));
      } else {
        uint8_t* const to = a.out + (int64_t)(base + (uint64_t)tr) * a.row_bytes;
        store_half<DT>(f, to, strip_col + c[0], a.C);
        store_half<DT>(f + 4, to, strip_col + c[1], a.C);
      }
    }
  }
  if constexpr (kSum) {
    const int cols = a.T * kChunkCols;  // of the strip
    if (tr < a.R)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) s_sum[tr * cols + c[j >> 2] + (j & 3)] = acc[j];
    __syncthreads();
    for (int at = threadIdx.x; at < cols && at < width; at += blockDim.x) {
      float sum = 0.f;
      for (int r = 0; r < a.R; ++r) sum += s_sum[r * cols + at];
      a.partial[(int64_t)blockIdx.x * a.C + strip_col + at] = sum;
    }
  }
}

// Workgroups that stay for many rows: those that sum columns, whose number is
// also that of the partial sums to write and to add (524288 x 768 bf16: 479 us
// with 1024, 486 with 2048, 513 with 4096, 570 with 768; without sums, a
// workgroup for every four rows a thread, 410), and those that fill a table (309
// with 2048, 329 with 1024).
constexpr int kSumBlocks = 1024, kTableBlocks = 2048;

// Elements from which the forward's table pays (50176 x 512: 22.8 us, without it 33.9; 8192 x 512 7.2 and 6.9).
constexpr int64_t kTableElements = 1ll << 22;

// 2^16 strips of 2^11 columns: what the grid's second dimension holds.
constexpr int64_t kDropMaxColumns = 1ll << 27;

struct DropPlan {
  int32_t T, R, strips;
  int64_t blocks;  // row slabs
};

// T chunk columns by R rows of threads; column strips where a row has more chunks than a workgroup threads.
DropPlan drop_plan(int64_t rows, int C, bool pieces, int64_t stay) {
  DropPlan p;
  const int chunks = (C - 1) / kChunkCols + 1;
  p.strips = (chunks - 1) / kDropThreads + 1;
  p.T = (chunks - 1) / p.strips + 1;
  p.T += pieces ? p.T & 1 : 0;  // lanes of a row in pairs
  p.R = kDropThreads / p.T;
  const int64_t per_block = (int64_t)p.R * kDropRows;
  p.blocks = (rows + per_block - 1) / per_block;
  // without a number, what a grid dimension of fewer than 2^32 threads holds
  const int64_t most = stay > 0 ? (stay + p.strips - 1) / p.strips : (1ll << 22);
  if (p.blocks > most) p.blocks = most;
  return p;
}

// Whether a call takes its GELU factors from a table.
bool drop_table(int op, int dtype, int64_t rows, int64_t C, bool vec) {
  return op == kGeluFwd && dtype == TERRA_DTYPE_BF16 && vec && rows * C >= kTableElements;
}

// How a call's rows are aligned: the bits that any of its addresses and row strides has set.
struct DropAlignment {
  uintptr_t bits = 0;
  int64_t C = 0;
  bool vec() const { return C % kChunkCols == 0 && bits % 16 == 0; }
  bool pairs() const { return C % 2 == 0 && bits % 4 == 0; }
};

template <int kOp, int DT>
void launch_drop(DropParams a, const DropAlignment& al, hipStream_t s) {
  const bool vec = al.vec(), table = drop_table(kOp, DT, a.rows, a.C, vec);
  const DropPlan p = drop_plan(a.rows, a.C, DT == TERRA_DTYPE_F32, table ? kTableBlocks : (kOp == kGeluBwdSum ? kSumBlocks : 0));
  a.T = p.T;
  a.R = p.R;
  const dim3 grid((unsigned)p.blocks, (unsigned)p.strips);
  const int threads = (p.T * p.R + 63) / 64 * 64;
  if constexpr (kOp == kGeluFwd && DT == TERRA_DTYPE_BF16)
    if (table) return (void)(drop_kernel<kOp, DT, true, true, false><<<grid, threads, 0, s>>>(a));
  if (vec) return (void)(drop_kernel<kOp, DT, true, false, false><<<grid, threads, 0, s>>>(a));
  if constexpr (DT != TERRA_DTYPE_F32)
    if (al.pairs()) return (void)(drop_kernel<kOp, DT, false, false, true><<<grid, threads, 0, s>>>(a));
  drop_kernel<kOp, DT, false, false, false><<<grid, threads, 0, s>>>(a);
}

template <int kOp>
void dispatch_drop(int dtype, const DropParams& a, const DropAlignment& al, hipStream_t s) {
  if (dtype == TERRA_DTYPE_F32) launch_drop<kOp, TERRA_DTYPE_F32>(a, al, s);
  else if (dtype == TERRA_DTYPE_BF16) launch_drop<kOp, TERRA_DTYPE_BF16>(a, al, s);
  else launch_drop<kOp, TERRA_DTYPE_F16>(a, al, s);
}

// The checks that the three entry points share; fills all but the pointers of `a`.
int drop_prepare(int dtype, int64_t rows, int64_t C, int64_t in_stride, double p, const void* seed, uint32_t stream,
                 DropParams* a, DropAlignment* al) {
  if (dtype != TERRA_DTYPE_F32 && dtype != TERRA_DTYPE_BF16 && dtype != TERRA_DTYPE_F16)
    return fail(TERRA_ERR_DTYPE, "dropout supports f32, bf16 and f16 (got dtype %d)", dtype);
  if (rows < 0 || C <= 0) return fail(TERRA_ERR_SHAPE, "rows must be >= 0 and columns > 0");
  if (rows >= (1ll << 31) || C >= kDropMaxColumns)
    return fail(TERRA_ERR_SHAPE, "%lld rows of %lld columns: at most 2^31 - 1 rows of 2^27 - 1", (long long)rows, (long long)C);
  if (in_stride < C) return fail(TERRA_ERR_SHAPE, "the row stride %lld is below the %lld columns", (long long)in_stride, (long long)C);
  const int st = dropout_args(p, seed, stream, &a->drop);
  if (st != TERRA_OK) return st;
  const int elt = dtype_size(dtype);
  a->rows = (uint32_t)rows;
  a->C = (int32_t)C;
  a->row_bytes = C * elt;
  a->in_row_bytes = in_stride * elt;
  al->C = C;
  al->bits = (uintptr_t)a->in_row_bytes;
  return TERRA_OK;
}

int drop_pointers(int dtype, std::initializer_list<const void*> tensors, DropAlignment* al) {
  for (const void* p : tensors) {
    if (p == nullptr) return fail(TERRA_ERR_NULL, "a tensor is NULL");
    if ((uintptr_t)p % (uintptr_t)dtype_size(dtype) != 0) return fail(TERRA_ERR_ALIGN, "a tensor is not aligned to its elements");
    al->bits |= (uintptr_t)p;
  }
  return TERRA_OK;
}

int drop_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TERRA_OK : fail(TERRA_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

// Whether [p, p + bytes) and [q, q + more) meet.
bool meet(const void* p, int64_t bytes, const void* q, int64_t more) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return bytes > 0 && more > 0 && a < b + (uintptr_t)more && b < a + (uintptr_t)bytes;
}

}  // namespace
}  // namespace terra

using namespace terra;

extern "C" int terra_swin_dropout(const void* x, void* y, int dtype, int64_t rows, int64_t columns, int64_t x_stride,
                                  double p, const void* seed, uint32_t stream_id, void* stream) {
  clear_error();
  DropParams a = {};
  DropAlignment al;
  int st = drop_prepare(dtype, rows, columns, x_stride, p, seed, stream_id, &a, &al);
  if (st != TERRA_OK || rows == 0) return st;
  if ((st = drop_pointers(dtype, {x, y}, &al)) != TERRA_OK) return st;
  if (!(x == y && x_stride == columns) &&
      meet(x, (rows - 1) * a.in_row_bytes + a.row_bytes, y, rows * a.row_bytes))
    return fail(TERRA_ERR_SHAPE, "y may be x itself (of packed rows) and must not overlap it otherwise");
  a.in = (const uint8_t*)x;
  a.out = (uint8_t*)y;
  dispatch_drop<kDropout>(dtype, a, al, (hipStream_t)stream);
  return drop_launched("terra_swin_dropout");
}

extern "C" int terra_swin_gelu_dropout(const void* h, void* a_out, int dtype, int64_t rows, int64_t columns, double p,
                                       const void* seed, uint32_t stream_id, void* stream) {
  clear_error();
  DropParams a = {};
  DropAlignment al;
  int st = drop_prepare(dtype, rows, columns, columns, p, seed, stream_id, &a, &al);
  if (st != TERRA_OK || rows == 0) return st;
  if ((st = drop_pointers(dtype, {h, a_out}, &al)) != TERRA_OK) return st;
  if (h != a_out && meet(h, rows * a.row_bytes, a_out, rows * a.row_bytes))
    return fail(TERRA_ERR_SHAPE, "a may be h itself and must not overlap it otherwise");
  a.in = (const uint8_t*)h;
  a.out = (uint8_t*)a_out;
  dispatch_drop<kGeluFwd>(dtype, a, al, (hipStream_t)stream);
  return drop_launched("terra_swin_gelu_dropout");
}

extern "C" int terra_swin_gelu_dropout_workspace(int64_t rows, int64_t columns) {
  clear_error();
  if (rows < 0 || columns <= 0 || rows >= (1ll << 31) || columns >= kDropMaxColumns)
    return fail(TERRA_ERR_SHAPE, "at most 2^31 - 1 rows of 1 to 2^27 - 1 columns");
  return rows == 0 ? 0 : (int)(drop_plan(rows, (int)columns, true, kSumBlocks).blocks * columns);
}

extern "C" int terra_swin_gelu_dropout_bwd(const void* da, const void* h, void* dh, int dtype, int64_t rows,
                                           int64_t columns, double p, const void* seed, uint32_t stream_id,
                                           float* column_sums, float* workspace, void* stream) {
  clear_error();
  DropParams a = {};
  DropAlignment al;
  int st = drop_prepare(dtype, rows, columns, columns, p, seed, stream_id, &a, &al);
  if (st != TERRA_OK) return st;
  if (((uintptr_t)column_sums & 3u) != 0 || ((uintptr_t)workspace & 3u) != 0)
    return fail(TERRA_ERR_ALIGN, "column_sums and workspace must be 4-byte aligned");
  hipStream_t s = (hipStream_t)stream;
  SumJobs jobs = {};
  jobs.C = (int32_t)columns;
  if (rows == 0) {  // the sums of no rows
    if (column_sums == nullptr) return TERRA_OK;
    jobs.job[0] = {column_sums, column_sums, 0, 0, 1};
    launch_sums(jobs, 1, s);
    return drop_launched("terra_swin_gelu_dropout_bwd");
  }
  if ((st = drop_pointers(dtype, {da, h, dh}, &al)) != TERRA_OK) return st;
  if (column_sums != nullptr && workspace == nullptr) return fail(TERRA_ERR_NULL, "column sums need a workspace");
  const int64_t bytes = rows * a.row_bytes;
  if ((da != dh && meet(da, bytes, dh, bytes)) || (h != dh && meet(h, bytes, dh, bytes)))
    return fail(TERRA_ERR_SHAPE, "dh may be da or h itself and must not overlap them otherwise");
  a.in = (const uint8_t*)da;
  a.h = (const uint8_t*)h;
  a.out = (uint8_t*)dh;
  a.partial = workspace;
  if (column_sums == nullptr) {
    dispatch_drop<kGeluBwd>(dtype, a, al, s);
  } else {
    dispatch_drop<kGeluBwdSum>(dtype, a, al, s);
    jobs.job[0] = {workspace, column_sums, columns, (int32_t)drop_plan(rows, (int)columns, dtype == TERRA_DTYPE_F32, kSumBlocks).blocks, 1};
    launch_sums(jobs, 1, s);
  }
  return drop_launched("terra_swin_gelu_dropout_bwd");
}
