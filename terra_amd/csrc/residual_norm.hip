// Entry points of the end of a half-block (residual_norm.h): argument checks,
// the backward's grid and workspace, and the choice of kernels by type.
#include "residual_norm.h"

namespace terra {
namespace {

// A tensor of the call: how far it reaches, for the overlap checks.
struct Span {
  const void* p;
  int64_t bytes;
  const char* name;
};

int check_spans(std::initializer_list<Span> in, std::initializer_list<Span> out) {
  for (const Span* o = out.begin(); o != out.end(); ++o) {
    if (o->p == nullptr) continue;
    auto meets = [&](const Span& s) {
      const uintptr_t a = (uintptr_t)o->p, b = (uintptr_t)s.p;
      return s.p != nullptr && s.bytes > 0 && o->bytes > 0 && a < b + (uintptr_t)s.bytes && b < a + (uintptr_t)o->bytes;
    };
    for (const Span& s : in)
      if (meets(s)) return fail(TERRA_ERR_SHAPE, "%s must not overlap %s", o->name, s.name);
    for (const Span* q = out.begin(); q != o; ++q)
      if (meets(*q)) return fail(TERRA_ERR_SHAPE, "%s must not overlap %s", o->name, q->name);
  }
  return TERRA_OK;
}

// How a call's rows are aligned: the bits that any of its addresses and row strides has set.
struct Alignment {
  uintptr_t bits = 0;
  int C = 0;
  bool vec() const { return C % kChunkCols == 0 && bits % 16 == 0; }
  bool pairs() const { return C % 2 == 0 && bits % 4 == 0; }
};

// Checks the descriptor; fills the sizes of `a` and `al`.  h_rows: rows of h.
int prepare(const terra_swin_residual_norm_desc* d, TailArgs* a, Alignment* al, int64_t* h_rows) {
  if (d == nullptr) return fail(TERRA_ERR_NULL, "desc is NULL");
  const int h = d->h_dtype, x = d->x_dtype;
  const bool half = h == TERRA_DTYPE_BF16 || h == TERRA_DTYPE_F16;
  if (!((half && (x == h || x == TERRA_DTYPE_F32)) || (h == TERRA_DTYPE_F32 && x == TERRA_DTYPE_F32)))
    return fail(TERRA_ERR_DTYPE, "h is bf16, f16 or f32 and x of h's dtype or f32 (got %d and %d)", h, x);
  if (d->rows < 0 || d->channels <= 0) return fail(TERRA_ERR_SHAPE, "rows must be >= 0 and channels > 0");
  if (d->channels > kTailMaxChannels)
    return fail(TERRA_ERR_UNSUPPORTED, "rows of up to %d channels (got %d)", kTailMaxChannels, d->channels);
  if (d->rows >= (1ll << 31)) return fail(TERRA_ERR_SHAPE, "%lld rows: at most 2^31 - 1", (long long)d->rows);
  for (int kind : {d->post_norm, d->next_norm})
    if (kind != TERRA_NORM_NONE && kind != TERRA_NORM_LAYER && kind != TERRA_NORM_RMS)
      return fail(TERRA_ERR_SHAPE, "unknown norm %d", kind);
  if (d->gate_rows < 0 || d->gate_rows >= (1ll << 31) || (d->gate_rows > 1 && d->rows % d->gate_rows != 0))
    return fail(TERRA_ERR_SHAPE, "%lld rows are not a whole number for each of %lld gate rows", (long long)d->rows,
                (long long)d->gate_rows);
  if (d->h_stride < d->channels || d->x_stride < d->channels)
    return fail(TERRA_ERR_SHAPE, "a row stride is below the %d channels", d->channels);
  a->rows = (uint32_t)d->rows;
  a->C = d->channels;
  a->flags = (d->post_norm != TERRA_NORM_NONE ? kTailPost : 0u) | (d->post_norm == TERRA_NORM_LAYER ? kTailPostLayer : 0u) |
             (d->next_norm != TERRA_NORM_NONE ? kTailNext : 0u) | (d->next_norm == TERRA_NORM_LAYER ? kTailNextLayer : 0u);
  a->post_eps = d->post_eps;
  a->next_eps = d->next_eps;
  a->alpha = d->residual_scale;
  a->inv_c = 1.f / (float)d->channels;
  // As many gate rows as rows are one each, whatever their number; the count fits 32 bits as the rows do.
  a->gate_rows = d->rows > 0 ? (int32_t)d->gate_rows : 0;
  a->per_sample = a->gate_rows > 1 ? (uint32_t)(d->rows / d->gate_rows) : a->rows;
  a->h_row_bytes = d->h_stride * dtype_size(h);
  a->x_row_bytes = d->x_stride * dtype_size(x);
  al->C = d->channels;
  al->bits = (uintptr_t)a->h_row_bytes | (uintptr_t)a->x_row_bytes;
  *h_rows = d->rows;
  if (d->windows && d->rows > 0) {
    a->flags |= kTailWindows;
    const terra_swin_geom& q = d->geom;
    GeomDims dims;
    const int st = validate_geom(&q, &dims);
    if (st != TERRA_OK) return st;
    if (q.channels != d->channels || (int64_t)q.batch * q.height * q.width != d->rows)
      return fail(TERRA_ERR_SHAPE, "the geometry's grid is not the %lld rows of %d channels", (long long)d->rows, d->channels);
    *h_rows = (int64_t)q.batch * dims.nWe * q.window * q.window;
    if (dims.Hp >= (1ll << 31) || dims.Wp >= (1ll << 31) || dims.nWe >= (1ll << 31))
      return fail(TERRA_ERR_SHAPE, "the window frame is too large");
    WindowMap& m = a->map;
    m.Hp = (int32_t)dims.Hp;
    m.Wp = (int32_t)dims.Wp;
    m.shift_h = q.shift_h;
    m.shift_w = q.shift_w;
    m.pad_top = q.pad_top;
    m.pad_left = q.pad_left;
    m.row_begin = q.win_row_begin;
    m.rows = (int32_t)dims.rows;
    m.cols = (int32_t)dims.nWw;
    m.ws = q.window;
    m.valid_begin = q.valid_begin;
    m.valid_end = q.valid_end > 0 ? q.valid_end : 0;
    m.fd_W = FastDiv((uint32_t)q.width);
    m.fd_H = FastDiv((uint32_t)q.height);
    m.fd_ws = FastDiv((uint32_t)q.window);
  }
  return TERRA_OK;
}

// Workgroups: what fits the 256 compute units at once; slabs of the rows of a
// sample so that every workgroup has a unit, and rows enough for its groups.
TailBwdPlan tail_bwd_plan(uint32_t rows, int C, int gate_rows, int x_dtype, bool vec) {
  TailBwdPlan p;
  p.shape = tail_shape(C, tail_pieces(x_dtype), tail_bwd_most(x_dtype, vec));
  const uint32_t groups = (uint32_t)(tail_threads(p.shape.lanes) / p.shape.lanes);
  const uint32_t most = p.shape.lanes > 256 ? 512u / (uint32_t)p.shape.chunks : (p.shape.chunks > 1 ? 512u : 1024u);
  const uint32_t samples = gate_rows > 1 ? (uint32_t)gate_rows : 1u, per = rows / samples;
  uint32_t slabs = (most + samples - 1) / samples;
  const uint32_t useful = (per + groups - 1) / groups;
  if (slabs > useful) slabs = useful;
  p.slabs = slabs;
  p.units = p.slabs * samples;
  p.blocks = p.units < most ? p.units : most;
  return p;
}

// f of the launches for the call's types.
#define TERRA_TAIL_LAUNCHES(h, x)                                                                    \
  struct Launch_##h##_##x {                                                                          \
    static void fwd(const void* a, bool vec, hipStream_t s) { tail_fwd_##h##_##x(a, vec, s); }       \
    static void bwd(const void* a, const TailBwdPlan& p, bool vec, hipStream_t s) { tail_bwd_##h##_##x(a, p, vec, s); } \
  };
TERRA_TAIL_TYPES(TERRA_TAIL_LAUNCHES)

template <typename F>
void by_type(const terra_swin_residual_norm_desc* d, F f) {
  const bool f32 = d->x_dtype == TERRA_DTYPE_F32;
  if (d->h_dtype == TERRA_DTYPE_F32) f(Launch_f32_f32{});
  else if (d->h_dtype == TERRA_DTYPE_BF16) f32 ? f(Launch_bf16_f32{}) : f(Launch_bf16_bf16{});
  else f32 ? f(Launch_f16_f32{}) : f(Launch_f16_f16{});
}

// Alignment of a tensor's or a parameter's pointer; NULL where it may be left out.
int check_pointer(const void* p, int elt, const char* name, bool needed, Alignment* al) {
  if (p == nullptr) return needed ? fail(TERRA_ERR_NULL, "%s is NULL", name) : TERRA_OK;
  if ((uintptr_t)p % (uintptr_t)elt != 0) return fail(TERRA_ERR_ALIGN, "%s is not aligned to its elements", name);
  al->bits |= (uintptr_t)p;
  return TERRA_OK;
}

int64_t span_bytes(int64_t rows, int64_t row_bytes, int64_t packed) { return rows > 0 ? (rows - 1) * row_bytes + packed : 0; }

int launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TERRA_OK : fail(TERRA_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace
}  // namespace terra

using namespace terra;

#define TERRA_TRY(call)                    \
  do {                                     \
    const int st_ = (call);                \
    if (st_ != TERRA_OK) return st_;       \
  } while (0)

extern "C" int terra_swin_residual_norm(const void* h, const void* x, void* y, void* z,
                                        const terra_swin_residual_norm_desc* desc,
                                        const float* post_weight, const float* post_bias, const float* gate,
                                        const float* next_weight, const float* next_bias,
                                        const void* seed, void* stream) {
  clear_error();
  TailArgs a = {};
  Alignment al;
  int64_t h_rows = 0;
  TERRA_TRY(prepare(desc, &a, &al, &h_rows));
  TERRA_TRY(dropout_args(desc->p, seed, desc->stream_id, &a.drop));
  if (a.drop.threshold > 0) a.flags |= kTailDrop;
  if (a.rows == 0) return TERRA_OK;
  const int he = dtype_size(desc->h_dtype), xe = dtype_size(desc->x_dtype);
  TERRA_TRY(check_pointer(h, he, "h", true, &al));
  TERRA_TRY(check_pointer(x, xe, "x", true, &al));
  TERRA_TRY(check_pointer(y, xe, "y", true, &al));
  TERRA_TRY(check_pointer(z, he, "z", (a.flags & kTailNext) != 0, &al));
  TERRA_TRY(check_pointer(gate, 4, "gate", a.gate_rows > 0, &al));
  for (const float* p : {post_weight, post_bias, next_weight, next_bias})
    TERRA_TRY(check_pointer(p, 4, "a norm's parameter", false, &al));
  const int64_t C = a.C;
  if ((a.flags & kTailNext) == 0) z = nullptr;
  TERRA_TRY(check_spans({{h, span_bytes(h_rows, a.h_row_bytes, C * he), "h"}, {x, span_bytes(a.rows, a.x_row_bytes, C * xe), "x"}},
                        {{y, a.rows * C * xe, "y"}, {z, a.rows * C * he, "z"}}));
  a.h = (const uint8_t*)h;
  a.x = (const uint8_t*)x;
  a.y = (uint8_t*)y;
  a.z = (uint8_t*)z;
  if ((a.flags & kTailPost) != 0) a.pw = post_weight, a.pb = post_bias;
  if ((a.flags & kTailNext) != 0) a.nw = next_weight, a.nb = next_bias;
  a.gate = gate;
  hipStream_t s = (hipStream_t)stream;
  if (al.pairs()) a.flags |= kTailPairs;
  by_type(desc, [&](auto t) { t.fwd(&a, al.vec(), s); });
  return launched("terra_swin_residual_norm");
}

// fp32 values: the workgroups' sums of four vectors, then the gate's units
// where a sample has several.  At most 1024 workgroups and twice as many units,
// fewer where rows are wide: the count fits an int.
extern "C" int terra_swin_residual_norm_workspace(const terra_swin_residual_norm_desc* desc) {
  clear_error();
  TailArgs a = {};
  Alignment al;
  int64_t h_rows = 0;
  TERRA_TRY(prepare(desc, &a, &al, &h_rows));
  if (a.rows == 0) return 0;
  int most = 0;
  for (const bool vec : {false, true}) {  // which, the call's addresses say
    const TailBwdPlan p = tail_bwd_plan(a.rows, a.C, a.gate_rows, desc->x_dtype, vec);
    const int n = (int)(p.blocks * 4 * a.C + (a.gate_rows > 0 && p.slabs > 1 ? p.units * a.C : 0));
    most = n > most ? n : most;
  }
  return most;
}

extern "C" int terra_swin_residual_norm_bwd(const void* h, const void* x, const void* dy, const void* dz, void* dh, void* dx,
                                            const terra_swin_residual_norm_desc* desc,
                                            const float* post_weight, const float* post_bias, const float* gate,
                                            const float* next_weight, const void* seed,
                                            float* dpost_weight, float* dpost_bias, float* dgate,
                                            float* dnext_weight, float* dnext_bias, float* workspace, void* stream) {
  clear_error();
  TailArgs a = {};
  Alignment al;
  int64_t h_rows = 0;
  TERRA_TRY(prepare(desc, &a, &al, &h_rows));
  TERRA_TRY(dropout_args(desc->p, seed, desc->stream_id, &a.drop));
  if (a.drop.threshold > 0) a.flags |= kTailDrop;
  const int he = dtype_size(desc->h_dtype), xe = dtype_size(desc->x_dtype);
  Alignment ignored;
  for (const float* p : {(const float*)dpost_weight, (const float*)dpost_bias, (const float*)dgate,
                         (const float*)dnext_weight, (const float*)dnext_bias, (const float*)workspace})
    TERRA_TRY(check_pointer(p, 4, "a parameter's gradient or the workspace", false, &ignored));
  if ((a.flags & kTailPost) == 0 && (dpost_weight != nullptr || dpost_bias != nullptr))
    return fail(TERRA_ERR_SHAPE, "gradients of a post-norm that the call has not");
  if ((a.flags & kTailNext) == 0 && (dz != nullptr || dnext_weight != nullptr || dnext_bias != nullptr))
    return fail(TERRA_ERR_SHAPE, "gradients of a next norm that the call has not");
  if (dgate != nullptr && desc->gate_rows == 0) return fail(TERRA_ERR_SHAPE, "the gradient of a gate that the call has not");
  hipStream_t s = (hipStream_t)stream;
  SumJobs jobs = {};
  jobs.C = a.C;
  int n = 0;
  if (a.rows == 0) {  // sums of no rows
    for (float* p : {dpost_weight, dpost_bias, dnext_weight, dnext_bias})
      if (p != nullptr) jobs.job[n++] = {p, p, 0, 0, 1};
    if (dgate != nullptr) jobs.job[n++] = {dgate, dgate, 0, 0, (int32_t)desc->gate_rows};
    if (n > 0) launch_sums(jobs, n, s);
    return launched("terra_swin_residual_norm_bwd");
  }
  TERRA_TRY(check_pointer(h, he, "h", true, &al));
  TERRA_TRY(check_pointer(x, xe, "x", true, &al));
  TERRA_TRY(check_pointer(dy, xe, "dy", false, &al));
  TERRA_TRY(check_pointer(dz, he, "dz", false, &al));
  TERRA_TRY(check_pointer(dh, he, "dh", true, &al));
  TERRA_TRY(check_pointer(dx, xe, "dx", true, &al));
  TERRA_TRY(check_pointer(gate, 4, "gate", a.gate_rows > 0, &al));
  for (const float* p : {post_weight, post_bias, next_weight})
    TERRA_TRY(check_pointer(p, 4, "a norm's parameter", false, &al));
  const bool sums = dpost_weight != nullptr || dpost_bias != nullptr || dnext_weight != nullptr || dnext_bias != nullptr;
  if ((sums || dgate != nullptr) && workspace == nullptr) return fail(TERRA_ERR_NULL, "parameter gradients need a workspace");
  const int64_t C = a.C;
  TERRA_TRY(check_spans({{h, span_bytes(h_rows, a.h_row_bytes, C * he), "h"}, {x, span_bytes(a.rows, a.x_row_bytes, C * xe), "x"},
                         {dy, a.rows * C * xe, "dy"}, {dz, a.rows * C * he, "dz"}},
                        {{dh, h_rows * C * he, "dh"}, {dx, a.rows * C * xe, "dx"}}));
  a.h = (const uint8_t*)h;
  a.x = (const uint8_t*)x;
  a.dy = (const uint8_t*)dy;
  a.dz = (const uint8_t*)dz;
  a.dh = (uint8_t*)dh;
  a.dx = (uint8_t*)dx;
  if ((a.flags & kTailPost) != 0) a.pw = post_weight, a.pb = post_bias;
  if ((a.flags & kTailNext) != 0) a.nw = next_weight;
  if (dz == nullptr) a.flags &= ~kTailNext;
  if (dy != nullptr) a.flags |= kTailDy;
  a.gate = gate;
  if (al.pairs()) a.flags |= kTailPairs;
  const TailBwdPlan p = tail_bwd_plan(a.rows, a.C, a.gate_rows, desc->x_dtype, al.vec());
  a.slabs = p.slabs;
  a.units = p.units;
  a.partial = sums ? workspace : nullptr;
  a.branch_sums = dpost_weight != nullptr || dpost_bias != nullptr || dgate != nullptr;
  // One slab a sample: the unit's sums are the gate's gradient itself.
  const bool direct = dgate != nullptr && p.slabs == 1;
  float* units = workspace + (int64_t)p.blocks * 4 * C;
  a.gate_partial = dgate == nullptr ? nullptr : (direct ? dgate : units);
  by_type(desc, [&](auto t) { t.bwd(&a, p, al.vec(), s); });
  float* dst[4] = {dpost_weight, dpost_bias, dnext_weight, dnext_bias};
  for (int i = 0; i < 4; ++i)
    if (dst[i] != nullptr) jobs.job[n++] = {workspace + i * C, dst[i], 4 * C, (int32_t)p.blocks, 1};
  if (dgate != nullptr && !direct)
    jobs.job[n++] = {units, dgate, C, (int32_t)p.slabs, a.gate_rows > 1 ? a.gate_rows : 1};
  if (n > 0) launch_sums(jobs, n, s);
  return launched("terra_swin_residual_norm_bwd");
}
