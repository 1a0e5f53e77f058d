// Entry points of the norms over rows (layer_norm.h).
#include "layer_norm.h"

#include <initializer_list>

namespace terra {
namespace {

constexpr int kNormMaxChannels = 1 << 24;

struct NormAlignment {
  uintptr_t bits = 0;
  int C = 0;
  bool packed = false;       // x's rows follow each other
  uintptr_t pointers = 0;    // the bits of the addresses alone
  bool vec() const { return C % kChunkCols == 0 && bits % 16 == 0; }
  bool pairs() const { return C % 2 == 0 && bits % 4 == 0; }
  bool flat() const { return !vec() && packed && pointers % 16 == 0; }
};

bool is_float(int dtype) { return dtype == TERRA_DTYPE_F32 || dtype == TERRA_DTYPE_BF16 || dtype == TERRA_DTYPE_F16; }

// Checks the descriptor; fills what it says of `a` and `al`.
int norm_prepare(const terra_swin_layer_norm_desc* d, NormArgs* a, NormAlignment* al) {
  if (d == nullptr) return fail(TERRA_ERR_NULL, "desc is NULL");
  const int x = d->x_dtype, y = d->y_dtype;
  if (!is_float(x) || !is_float(y) || !is_float(d->param_dtype) || (x != y && x != TERRA_DTYPE_F32 && y != TERRA_DTYPE_F32))
    return fail(TERRA_ERR_DTYPE, "x, y and the parameters are f32, bf16 or f16, y of x's dtype unless one is f32 (got %d, %d, %d)",
                x, y, d->param_dtype);
  if (d->rows < 0 || d->channels <= 0) return fail(TERRA_ERR_SHAPE, "rows must be >= 0 and channels > 0");
  if (d->channels > kNormMaxChannels)
    return fail(TERRA_ERR_UNSUPPORTED, "rows of up to %d channels (got %d)", kNormMaxChannels, d->channels);
  if (d->rows >= (1ll << 31)) return fail(TERRA_ERR_SHAPE, "%lld rows: at most 2^31 - 1", (long long)d->rows);
  if (d->norm != TERRA_NORM_LAYER && d->norm != TERRA_NORM_RMS) return fail(TERRA_ERR_SHAPE, "unknown norm %d", d->norm);
  if (d->inner <= 0 || d->inner >= (1ll << 31)) return fail(TERRA_ERR_SHAPE, "inner must be in [1, 2^31) (got %lld)", (long long)d->inner);
  if (d->outer_stride < 0 || d->inner_stride < 0 || d->outer_stride >= (1ll << 40) || d->inner_stride >= (1ll << 40))
    return fail(TERRA_ERR_SHAPE, "row strides must be in [0, 2^40)");
  if (!(d->eps >= 0.f)) return fail(TERRA_ERR_SHAPE, "eps must be >= 0 (got %g)", (double)d->eps);
  const int elt = dtype_size(x);
  a->rows = (uint32_t)d->rows;
  a->C = d->channels;
  a->inner = FastDiv((uint32_t)d->inner);
  a->outer_bytes = d->outer_stride * elt;
  a->step_bytes = d->inner_stride * elt;
  a->param_dtype = d->param_dtype;
  a->layer = d->norm == TERRA_NORM_LAYER;
  a->eps = d->eps;
  a->inv_c = 1.f / (float)d->channels;
  al->C = a->C;
  al->packed = (d->rows <= 1 || (d->inner_stride == d->channels || d->inner == 1)) &&
               (d->rows <= d->inner || d->outer_stride == d->inner * d->channels);
  al->bits = (d->rows > d->inner ? (uintptr_t)a->outer_bytes : 0) | (d->inner > 1 ? (uintptr_t)a->step_bytes : 0);
  return TERRA_OK;
}

int norm_pointer(const void* p, int dtype, const char* name, bool needed, NormAlignment* al) {
  if (p == nullptr) return needed ? fail(TERRA_ERR_NULL, "%s is NULL", name) : TERRA_OK;
  if ((uintptr_t)p % (uintptr_t)dtype_size(dtype) != 0) return fail(TERRA_ERR_ALIGN, "%s is not aligned to its elements", name);
  if (al != nullptr) al->bits |= (uintptr_t)p, al->pointers |= (uintptr_t)p;
  return TERRA_OK;
}

// Bytes from the first row of x to the end of its last one.
int64_t x_span(const terra_swin_layer_norm_desc* d) {
  if (d->rows == 0) return 0;
  const int64_t outer = (d->rows - 1) / d->inner, inner = d->rows < d->inner ? d->rows - 1 : d->inner - 1;
  return (outer * d->outer_stride + inner * d->inner_stride + d->channels) * dtype_size(d->x_dtype);
}

bool norm_meet(const void* p, int64_t bytes, const void* q, int64_t more) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p != nullptr && q != nullptr && bytes > 0 && more > 0 && a < b + (uintptr_t)more && b < a + (uintptr_t)bytes;
}

constexpr int kNormHeld = 16384;  // channels of rows that are held in registers

// How many lanes and chunks hold a row.  Waves rather than workgroups as far as the registers
// go: what its lanes add up needs no barrier (39168 x 4096 bf16, forward: 118 us, as 512 lanes
// of one chunk 135; 78336 x 2048: 108 and 143).  The backward, with two sums for each column
// and two rows, goes so far as four chunks (78336 x 2048: 156 us, as 256 lanes 167; 39168 x 4096 as
// 256 lanes of two 161, as waves of eight 175); rows that are not aligned or that have fp32 in them as far as two
// where a few lanes hold them.  As few lanes as chunks where a row has at most eight: the heads of a packed q | k | v.
constexpr TailShape norm_shape(int C, bool pieces, bool vec, bool backward) {
  const int n = (C + kChunkCols - 1) / kChunkCols;
  if (n <= 8) return {n <= 2 ? 2 : n <= 4 ? 4 : 8, 1};
  if (n > 1024) return {1024, 2};
  if (n > 512) return {512, 2};
  if (n > 256) return backward ? TailShape{256, 2} : TailShape{64, 8};
  if (n > 128) return {64, 4};
  return tail_shape(C, pieces, backward && (pieces || !vec) ? 2 : 3);
}

// The same for rows that are read by the aligned chunks of the tensor, a chunk more than C takes where the
// row begins in one.  Parameters stand in registers too: one to three chunks a lane, up to four where waves can hold the
// row so.  Three where two would leave many lanes idle (60 million elements, bf16 backward: 514 by 32 lanes of
// three 83 us, by 64 of two 108; 1030 by 64 of three 82, by 64 of four 141, by 256 of one 163).
constexpr TailShape flat_shape(int C, int chunk) {
  const int n = (C + chunk - 1 + kChunkCols - 1) / kChunkCols;
  if (n <= 16) return {n <= 8 ? 8 : 16, 1};
  for (int lanes = 8; lanes <= 32; lanes *= 2) {
    if (n <= 2 * lanes) return {lanes, 2};
    if (n <= 3 * lanes) return {lanes, 3};
  }
  if (n <= 256) return {64, n <= 128 ? 2 : n <= 192 ? 3 : 4};
  return {n <= 512 ? 256 : n <= 1024 ? 512 : 1024, 2};
}

// Every row that is held has a shape that holds it, among those that the launches know (layer_norm_kernels.h, where
// eight lanes of three chunks have no kernel that accesses fp32 by pieces).
constexpr bool norm_shape_known(TailShape s, bool pieces, bool backward) {
  switch (s.lanes * 10 + s.chunks) {
    case 21: case 41: case 81: case 161: case 162: case 163: case 322: case 323: case 642: case 644: case 5122: case 10242: return true;
    case 83: return !pieces;
    case 648: return !backward;
    case 2562: return backward;
    default: return false;
  }
}
constexpr bool flat_shape_known(TailShape s) {
  switch (s.lanes * 10 + s.chunks) {
    case 81: case 83: case 161: case 162: case 163: case 322: case 323: case 642: case 643: case 644: case 2562: case 5122:
    case 10242: return true;
    default: return false;
  }
}
constexpr bool norm_shapes_hold() {
  for (int n = 1; n <= kNormHeld / kChunkCols; ++n)  // a shape goes by the chunks of a row
    for (int options = 0; options < 8; ++options) {
      const bool pieces = options & 1, backward = options & 4;
      const TailShape s = norm_shape(n * kChunkCols, pieces, options & 2, backward);
      if (s.lanes * s.chunks < n || !norm_shape_known(s, pieces, backward)) return false;
    }
  return true;
}
constexpr bool flat_shapes_hold() {
  for (int n = 2; n <= kNormHeld / kChunkCols; ++n)
    for (int chunk = 4; chunk <= kChunkCols; chunk += 4) {  // of the widest row that touches n chunks
      const TailShape s = flat_shape(n * kChunkCols - chunk + 1, chunk);
      if (s.lanes * s.chunks < n || !flat_shape_known(s)) return false;
    }
  return true;
}
static_assert(norm_shapes_hold(), "a row without a shape that holds it");
static_assert(flat_shapes_hold(), "a packed row without a shape that holds it");

// Whether packed rows that are not whole chunks are read by the tensor's aligned chunks, or by columns (16-bit ones by pairs
// where those stand aligned).  60 million elements, by chunks and by columns, us: 1001 bf16 forward 57, 92, backward
// 76, 134; 1030 bf16 59, 73 and 82, 136; 1030 fp32 100, 119 and 135, 219; 4097 fp32 96, 129 and 144, 199.  Narrow
// rows share their chunks with too many neighbours: 17 fp32 157, 101 and 244, 186; 50 bf16 forward 69, 64, 61 bf16
// 84, 71, but 33 bf16 backward 115, 186.
bool norm_flat(int C, bool pieces, bool backward) {
  const int chunk = pieces ? 4 : kChunkCols;
  if (C + chunk - 1 > kNormHeld) return false;
  if (backward) return C >= 32;
  return C >= 64;
}

// Workgroups of the sums over rows, at most what fits the 256 compute units at once (524288 x 192
// bf16: 512 workgroups 84 us, 1024 93; with four chunks a lane one wave a SIMD does).
NormPlan norm_plan(uint32_t rows, int C, bool pieces, bool vec, bool flat, bool backward) {
  NormPlan p = {};
  p.flat = flat && norm_flat(C, pieces, backward);
  p.held = !p.flat && C <= kNormHeld;
  if (p.flat || p.held) {
    p.shape = p.flat ? flat_shape(C, pieces ? 4 : kChunkCols) : norm_shape(C, pieces, vec, backward);
    const uint32_t groups = (uint32_t)(tail_threads(p.shape.lanes) / p.shape.lanes), useful = (rows + groups - 1) / groups;
    const uint32_t most = p.shape.chunks >= 4 || p.shape.lanes > 512 ? 256u : p.shape.lanes <= 16 && p.shape.chunks == 1 ? 1024u : 512u;
    p.parts = useful < most ? useful : most;
    if (p.flat) p.parts = (p.parts + 7) / 8 * 8;  // rows of a group: a multiple of eight apart
    return p;
  }
  const uint32_t strips = (uint32_t)((C + 511) / 512), most = strips < 1024 ? 1024 / strips : 1, useful = (rows + 31) / 32;
  p.parts = useful < most ? useful : most;
  return p;
}

bool norm_by_pieces(const terra_swin_layer_norm_desc* d) { return d->x_dtype == TERRA_DTYPE_F32 || d->y_dtype == TERRA_DTYPE_F32; }

// dst[c] = sum over i < parts of partial[i][which][c], in fp64, in the parameters' type.
struct FinishArgs {
  const float* partial;
  void* dst[2];
  int32_t parts, C, dtype;
};
constexpr int kFinishThreads = 1024, kFinishCols = 16, kFinishParts = kFinishThreads / kFinishCols;

__global__ __launch_bounds__(kFinishThreads) void norm_finish_kernel(const FinishArgs a) {
  __shared__ double s[kFinishParts][kFinishCols];
  const int which = blockIdx.y, lane = threadIdx.x % kFinishCols, part = threadIdx.x / kFinishCols;
  const int c = blockIdx.x * kFinishCols + lane;
  double sum = 0.0;
  const float* src = a.partial + (int64_t)which * a.C + (c < a.C ? c : 0);
  constexpr int kAhead = 8;
  for (int i = part; i < a.parts; i += kAhead * kFinishParts) {
    float v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = i + u * kFinishParts;
      v[u] = src[(int64_t)(at < a.parts ? at : i) * 2 * a.C];
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) sum += i + u * kFinishParts < a.parts ? (double)v[u] : 0.0;
  }
  s[part][lane] = sum;
  __syncthreads();
  for (int half = kFinishParts / 2; half > 0; half /= 2) {
    if (part < half) s[part][lane] = sum += s[part + half][lane];
    __syncthreads();
  }
  if (part != 0 || c >= a.C || a.dst[which] == nullptr) return;
  const float v = (float)sum;
  if (a.dtype == TERRA_DTYPE_F32) reinterpret_cast<float*>(a.dst[which])[c] = v;
  else if (a.dtype == TERRA_DTYPE_BF16) reinterpret_cast<uint16_t*>(a.dst[which])[c] = f32_to_bf16_bits(v);
  else reinterpret_cast<uint16_t*>(a.dst[which])[c] = __half_as_ushort(__float2half_rn(v));
}

int norm_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TERRA_OK : fail(TERRA_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

#define TERRA_NORM_CASE(x, y) \
  if (xd == kNorm_##x && yd == kNorm_##y) return backward ? norm_bwd_##x##_##y(&a, p, vec, pairs, s) : norm_fwd_##x##_##y(&a, p, vec, pairs, s);
constexpr int kNorm_f32 = TERRA_DTYPE_F32, kNorm_bf16 = TERRA_DTYPE_BF16, kNorm_f16 = TERRA_DTYPE_F16;
void norm_launch(bool backward, int xd, int yd, const NormArgs& a, const NormPlan& p, const NormAlignment& al, hipStream_t s) {
  const bool vec = al.vec(), pairs = al.pairs();
  TERRA_NORM_TYPES(TERRA_NORM_CASE)
}

}  // namespace
}  // namespace terra

using namespace terra;

#define TERRA_TRY(call)                    \
  do {                                     \
    const int st_ = (call);                \
    if (st_ != TERRA_OK) return st_;       \
  } while (0)

extern "C" int terra_swin_layer_norm(const void* x, void* y, const terra_swin_layer_norm_desc* desc, const void* weight,
                                     const void* bias, float* statistics, void* stream) {
  clear_error();
  NormArgs a = {};
  NormAlignment al;
  TERRA_TRY(norm_prepare(desc, &a, &al));
  if (a.rows == 0) return TERRA_OK;
  TERRA_TRY(norm_pointer(x, desc->x_dtype, "x", true, &al));
  TERRA_TRY(norm_pointer(y, desc->y_dtype, "y", true, &al));
  TERRA_TRY(norm_pointer(weight, desc->param_dtype, "the weight", false, nullptr));
  TERRA_TRY(norm_pointer(bias, desc->param_dtype, "the bias", false, nullptr));
  if (((uintptr_t)statistics & 7u) != 0) return fail(TERRA_ERR_ALIGN, "statistics must be 8-byte aligned");
  const int64_t out = (int64_t)a.rows * a.C * dtype_size(desc->y_dtype), span = x_span(desc);
  if (norm_meet(x, span, y, out)) return fail(TERRA_ERR_SHAPE, "y must not overlap x");
  if (norm_meet(statistics, (int64_t)a.rows * 8, x, span) || norm_meet(statistics, (int64_t)a.rows * 8, y, out))
    return fail(TERRA_ERR_SHAPE, "statistics must not overlap x or y");
  a.x = (const uint8_t*)x;
  a.y = (uint8_t*)y;
  a.w = weight;
  a.b = bias;
  a.statistics = (float2*)statistics;
  norm_launch(false, desc->x_dtype, desc->y_dtype, a,
              norm_plan(a.rows, a.C, norm_by_pieces(desc), al.vec(), al.flat(), false), al, (hipStream_t)stream);
  return norm_launched("terra_swin_layer_norm");
}

extern "C" int terra_swin_layer_norm_workspace(const terra_swin_layer_norm_desc* desc) {
  clear_error();
  NormArgs a = {};
  NormAlignment al;
  TERRA_TRY(norm_prepare(desc, &a, &al));
  if (a.rows == 0) return 0;
  int most = 0;
  for (const bool vec : {false, true})  // which, the call's addresses say
    for (const bool flat : {false, true}) {
      const int n = (int)norm_plan(a.rows, a.C, norm_by_pieces(desc), vec, flat && !vec, true).parts * 2 * a.C;
      most = n > most ? n : most;
    }
  return most;
}

extern "C" int terra_swin_layer_norm_bwd(const void* dy, const void* x, const float* statistics, void* dx,
                                         const terra_swin_layer_norm_desc* desc, const void* weight, void* dweight,
                                         void* dbias, float* workspace, void* stream) {
  clear_error();
  NormArgs a = {};
  NormAlignment al;
  TERRA_TRY(norm_prepare(desc, &a, &al));
  const int xd = desc->x_dtype, yd = desc->y_dtype;
  TERRA_TRY(norm_pointer(dweight, desc->param_dtype, "dweight", false, nullptr));
  TERRA_TRY(norm_pointer(dbias, desc->param_dtype, "dbias", false, nullptr));
  const bool sums = dweight != nullptr || dbias != nullptr;
  if (dx == nullptr && !sums) return TERRA_OK;
  FinishArgs f = {workspace, {dweight, dbias}, 0, a.C, desc->param_dtype};
  hipStream_t s = (hipStream_t)stream;
  const dim3 finish((unsigned)((a.C + kFinishCols - 1) / kFinishCols), 2);
  if (a.rows == 0) {  // the sums of no rows
    if (!sums) return TERRA_OK;
    norm_finish_kernel<<<finish, kFinishThreads, 0, s>>>(f);
    return norm_launched("terra_swin_layer_norm_bwd");
  }
  TERRA_TRY(norm_pointer(dy, yd, "dy", true, &al));
  TERRA_TRY(norm_pointer(x, xd, "x", true, &al));
  TERRA_TRY(norm_pointer(dx, xd, "dx", false, &al));
  TERRA_TRY(norm_pointer(weight, desc->param_dtype, "the weight", false, nullptr));
  if (statistics == nullptr) return fail(TERRA_ERR_NULL, "statistics are NULL");
  if (((uintptr_t)statistics & 7u) != 0) return fail(TERRA_ERR_ALIGN, "statistics must be 8-byte aligned");
  if (sums && workspace == nullptr) return fail(TERRA_ERR_NULL, "parameter gradients need a workspace");
  if (((uintptr_t)workspace & 3u) != 0) return fail(TERRA_ERR_ALIGN, "the workspace must be 4-byte aligned");
  const int64_t n = (int64_t)a.rows * a.C, in = n * dtype_size(yd), out = n * dtype_size(xd);
  if (norm_meet(dx, out, x, x_span(desc)) || norm_meet(dx, out, statistics, (int64_t)a.rows * 8) || norm_meet(dx, out, dy, in))
    return fail(TERRA_ERR_SHAPE, "dx must not overlap x, dy or the statistics");
  a.x = (const uint8_t*)x;
  a.dy = (const uint8_t*)dy;
  a.dx = (uint8_t*)dx;
  a.w = weight;
  a.statistics = (float2*)const_cast<float*>(statistics);
  const NormPlan p = norm_plan(a.rows, a.C, norm_by_pieces(desc), al.vec(), al.flat(), true);
  a.parts = p.parts;
  a.partial = sums ? workspace : nullptr;
  norm_launch(true, xd, yd, a, p, al, s);
  if (sums) {
    f.parts = (int32_t)p.parts;
    norm_finish_kernel<<<finish, kFinishThreads, 0, s>>>(f);
  }
  return norm_launched("terra_swin_layer_norm_bwd");
}
