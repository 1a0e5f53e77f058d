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
// Layout: a thread owns one chunk column and steps through rows, so column
// sums stay in its registers; a workgroup is T chunk columns by R rows.
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
// 4.4e-7 relative for h < 0, 1.7e-7 absolute), so the tail keeps its relative
// precision.  About 20 instructions, of which exp2 and the reciprocal go to the
// transcendental unit; erfcf and expf took three times as many.
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

template <int kOp>
__device__ __forceinline__ float drop_value(float v, float h) {
  if constexpr (kOp == kDropout) return v;
  else if constexpr (kOp == kGeluFwd) return v * gelu_factor(v);
  else return v * gelu_slope_of(h);
}

template <int kOp, int DT, bool kVec>
__global__ __launch_bounds__(kDropThreads) void drop_kernel(const DropParams a) {
  constexpr int kB = ChunkElt<DT>::kBytes;
  constexpr bool kBwd = kOp >= kGeluBwd;
  constexpr bool kSum = kOp == kGeluBwdSum;
  __shared__ float s_sum[kSum ? kDropThreads * kChunkCols : 1];
  const int tc = threadIdx.x % a.T, tr = threadIdx.x / a.T;
  const int chunk = blockIdx.y * a.T + tc, col = chunk * kChunkCols;
  const bool present = tr < a.R && col < a.C;
  const int64_t strip = (int64_t)blockIdx.y * a.T * kChunkCols * kB;  // bytes before this strip of columns
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
      v[i] = load_chunk<DT, kVec>(a.in + r * a.in_row_bytes, col, a.C, present);
      if constexpr (kBwd) hv[i] = load_chunk<DT, kVec>(a.h + r * a.row_bytes, col, a.C, present);
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
      float f[kChunkCols], g[kChunkCols];
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) {
        f[j] = chunk_value<DT>(v[i], j);
        if constexpr (kBwd) g[j] = chunk_value<DT>(hv[i], j);
      }
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) f[j] = drop_value<kOp>(f[j], kBwd ? g[j] : 0.f);
      if (a.drop.threshold > 0) {
        const ChunkDraws d = chunk_draws(seed, (uint32_t)chunk, (uint32_t)base + (uint32_t)tr, a.drop.stream);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) f[j] = kept(d, j, a.drop.threshold) ? f[j] * a.drop.scale : 0.f;
      }
      if constexpr (kSum)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) acc[j] += f[j];
      store_chunk<DT, kVec>(f, out, (uint32_t)((int64_t)tr * a.row_bytes) + (uint32_t)(tc * kChunkCols * kB), col, a.C);
    }
  }
  if constexpr (kSum) {
    const int width = a.T * kChunkCols;
    if (tr < a.R)
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) s_sum[tr * width + tc * kChunkCols + j] = acc[j];
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += blockDim.x) {
      const int out_col = blockIdx.y * width + c;
      if (out_col >= a.C) break;
      float sum = 0.f;
      for (int r = 0; r < a.R; ++r) sum += s_sum[r * width + c];
      a.partial[(int64_t)blockIdx.x * a.C + out_col] = sum;
    }
  }
}

// Workgroups that sum columns: about eight for each of the 256 compute units.
constexpr int kSumBlocks = 2048;

struct DropPlan {
  int32_t T, R, strips;
  int64_t blocks;  // row slabs
};

// T chunk columns by R rows of threads; column strips where a row has more chunks than a workgroup threads.
DropPlan drop_plan(int64_t rows, int C, bool sums) {
  DropPlan p;
  const int chunks = (C - 1) / kChunkCols + 1;
  p.strips = (chunks - 1) / kDropThreads + 1;
  p.T = (chunks - 1) / p.strips + 1;
  p.R = kDropThreads / p.T;
  const int64_t per_block = (int64_t)p.R * kDropRows;
  p.blocks = (rows + per_block - 1) / per_block;
  const int64_t most = sums ? (kSumBlocks + p.strips - 1) / p.strips : (1ll << 22);  // a grid dimension holds fewer than 2^32 threads
  if (p.blocks > most) p.blocks = most;
  return p;
}

template <int kOp, int DT>
void launch_drop(const DropParams& a, const DropPlan& p, bool vec, hipStream_t s) {
  const dim3 grid((unsigned)p.blocks, (unsigned)p.strips);
  const int threads = (p.T * p.R + 63) / 64 * 64;
  if (vec) drop_kernel<kOp, DT, true><<<grid, threads, 0, s>>>(a);
  else drop_kernel<kOp, DT, false><<<grid, threads, 0, s>>>(a);
}

template <int kOp>
void dispatch_drop(int dtype, const DropParams& a, const DropPlan& p, bool vec, hipStream_t s) {
  if (dtype == TERRA_DTYPE_F32) launch_drop<kOp, TERRA_DTYPE_F32>(a, p, vec, s);
  else if (dtype == TERRA_DTYPE_BF16) launch_drop<kOp, TERRA_DTYPE_BF16>(a, p, vec, s);
  else launch_drop<kOp, TERRA_DTYPE_F16>(a, p, vec, s);
}

// The checks that the three entry points share; fills all but the pointers of `a`.
int drop_prepare(int dtype, int64_t rows, int64_t C, int64_t in_stride, double p, const void* seed, uint32_t stream,
                 DropParams* a, bool* vec) {
  if (dtype != TERRA_DTYPE_F32 && dtype != TERRA_DTYPE_BF16 && dtype != TERRA_DTYPE_F16)
    return fail(TERRA_ERR_DTYPE, "dropout supports f32, bf16 and f16 (got dtype %d)", dtype);
  if (rows < 0 || C <= 0) return fail(TERRA_ERR_SHAPE, "rows must be >= 0 and columns > 0");
  if (rows >= (1ll << 31) || C >= (1ll << 24))
    return fail(TERRA_ERR_SHAPE, "%lld rows of %lld columns: at most 2^31 - 1 rows of 2^24 - 1", (long long)rows, (long long)C);
  if (in_stride < C) return fail(TERRA_ERR_SHAPE, "the row stride %lld is below the %lld columns", (long long)in_stride, (long long)C);
  const int st = dropout_args(p, seed, stream, &a->drop);
  if (st != TERRA_OK) return st;
  const int elt = dtype_size(dtype);
  a->rows = (uint32_t)rows;
  a->C = (int32_t)C;
  a->row_bytes = C * elt;
  a->in_row_bytes = in_stride * elt;
  *vec = C % kChunkCols == 0 && a->in_row_bytes % 16 == 0;
  return TERRA_OK;
}

int drop_pointers(int dtype, std::initializer_list<const void*> tensors, bool* vec) {
  for (const void* p : tensors) {
    if (p == nullptr) return fail(TERRA_ERR_NULL, "a tensor is NULL");
    if ((uintptr_t)p % (uintptr_t)dtype_size(dtype) != 0) return fail(TERRA_ERR_ALIGN, "a tensor is not aligned to its elements");
    if ((uintptr_t)p % 16 != 0) *vec = false;
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
  bool vec = false;
  int st = drop_prepare(dtype, rows, columns, x_stride, p, seed, stream_id, &a, &vec);
  if (st != TERRA_OK || rows == 0) return st;
  if ((st = drop_pointers(dtype, {x, y}, &vec)) != TERRA_OK) return st;
  if (!(x == y && x_stride == columns) &&
      meet(x, (rows - 1) * a.in_row_bytes + a.row_bytes, y, rows * a.row_bytes))
    return fail(TERRA_ERR_SHAPE, "y may be x itself (of packed rows) and must not overlap it otherwise");
  a.in = (const uint8_t*)x;
  a.out = (uint8_t*)y;
  const DropPlan plan = drop_plan(rows, (int)columns, false);
  a.T = plan.T;
  a.R = plan.R;
  dispatch_drop<kDropout>(dtype, a, plan, vec, (hipStream_t)stream);
  return drop_launched("terra_swin_dropout");
}

extern "C" int terra_swin_gelu_dropout(const void* h, void* a_out, int dtype, int64_t rows, int64_t columns, double p,
                                       const void* seed, uint32_t stream_id, void* stream) {
  clear_error();
  DropParams a = {};
  bool vec = false;
  int st = drop_prepare(dtype, rows, columns, columns, p, seed, stream_id, &a, &vec);
  if (st != TERRA_OK || rows == 0) return st;
  if ((st = drop_pointers(dtype, {h, a_out}, &vec)) != TERRA_OK) return st;
  if (h != a_out && meet(h, rows * a.row_bytes, a_out, rows * a.row_bytes))
    return fail(TERRA_ERR_SHAPE, "a may be h itself and must not overlap it otherwise");
  a.in = (const uint8_t*)h;
  a.out = (uint8_t*)a_out;
  const DropPlan plan = drop_plan(rows, (int)columns, false);
  a.T = plan.T;
  a.R = plan.R;
  dispatch_drop<kGeluFwd>(dtype, a, plan, vec, (hipStream_t)stream);
  return drop_launched("terra_swin_gelu_dropout");
}

extern "C" int terra_swin_gelu_dropout_workspace(int64_t rows, int64_t columns) {
  clear_error();
  if (rows < 0 || columns <= 0 || rows >= (1ll << 31) || columns >= (1ll << 24))
    return fail(TERRA_ERR_SHAPE, "at most 2^31 - 1 rows of 1 to 2^24 - 1 columns");
  return rows == 0 ? 0 : (int)(drop_plan(rows, (int)columns, true).blocks * columns);
}

extern "C" int terra_swin_gelu_dropout_bwd(const void* da, const void* h, void* dh, int dtype, int64_t rows,
                                           int64_t columns, double p, const void* seed, uint32_t stream_id,
                                           float* column_sums, float* workspace, void* stream) {
  clear_error();
  DropParams a = {};
  bool vec = false;
  int st = drop_prepare(dtype, rows, columns, columns, p, seed, stream_id, &a, &vec);
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
  if ((st = drop_pointers(dtype, {da, h, dh}, &vec)) != TERRA_OK) return st;
  if (column_sums != nullptr && workspace == nullptr) return fail(TERRA_ERR_NULL, "column sums need a workspace");
  const int64_t bytes = rows * a.row_bytes;
  if ((da != dh && meet(da, bytes, dh, bytes)) || (h != dh && meet(h, bytes, dh, bytes)))
    return fail(TERRA_ERR_SHAPE, "dh may be da or h itself and must not overlap them otherwise");
  a.in = (const uint8_t*)da;
  a.h = (const uint8_t*)h;
  a.out = (uint8_t*)dh;
  a.partial = workspace;
  const DropPlan plan = drop_plan(rows, (int)columns, column_sums != nullptr);
  a.T = plan.T;
  a.R = plan.R;
  if (column_sums == nullptr) {
    dispatch_drop<kGeluBwd>(dtype, a, plan, vec, s);
  } else {
    dispatch_drop<kGeluBwdSum>(dtype, a, plan, vec, s);
    jobs.job[0] = {workspace, column_sums, columns, (int32_t)plan.blocks, 1};
    launch_sums(jobs, 1, s);
  }
  return drop_launched("terra_swin_gelu_dropout_bwd");
}
