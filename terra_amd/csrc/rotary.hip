// Rotary positions: pairs (u, v) of a head's first `dim` elements turn by the
// angle t = 2 pi f position, f the turns a position of their rate:
//
//   u' = a (u cos t - v sin t),  v' = a (u sin t + v cos t)
//
// with the pairs (2i, 2i + 1) or (i, i + dim / 2); the backward is the same with
// -t, the rest of a head is copied.  The product f position is taken in 64 bits and
// brought to the nearest whole turn there: in 32 the angle of position 10^6 would be off by 0.06.
// The rotation is in fp32, rounded once.
//
// A thread has kP pairs of a token and goes through heads with them, so an angle's sine
// and cosine serve all of those.
#include "row_chunk.h"

#include <initializer_list>

namespace terra {
namespace {

struct RotaryArgs {
  const uint8_t* x;
  uint8_t* y;
  const void* positions;
  const double* turns;
  int64_t x_outer, x_inner, x_head, y_outer, y_inner, y_head;  // bytes
  FastDiv inner, position_tokens, lanes;  // lanes: threads of a token
  uint32_t tokens, per_block;             // tokens of a workgroup
  int32_t turned, items;                  // items of a token that are rotated, and all
  int32_t heads, per_thread;              // heads, of which a thread takes this many
  int32_t half;                           // dim / 2
  int32_t axes, per_axis;
  int32_t wide_positions;                 // 64-bit positions
  float amplitude, sign;
};

template <int DT> struct RotaryElt { typedef uint16_t type; };
template <> struct RotaryElt<TERRA_DTYPE_F32> { typedef uint32_t type; };

template <int DT>
__device__ __forceinline__ float rotary_value(typename RotaryElt<DT>::type v) {
  if constexpr (DT == TERRA_DTYPE_F32) return __uint_as_float(v);
  else if constexpr (DT == TERRA_DTYPE_BF16) return bf16_bits_to_f32(v);
  else return __half2float(__ushort_as_half(v));
}
template <int DT>
__device__ __forceinline__ typename RotaryElt<DT>::type rotary_round(float v) {
  if constexpr (DT == TERRA_DTYPE_F32) return __float_as_uint(v);
  else return (uint16_t)pack2<DT>(v, 0.f);
}

// kN elements that lie side by side, read or written as one access where aligned (kN elements of alignment).
template <int DT, int kN, bool kAligned>
struct RotaryRun {
  typedef typename RotaryElt<DT>::type Elt;
  Elt v[kN];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (kAligned) {
      typedef Elt vec __attribute__((ext_vector_type(kN)));
      const vec t = __builtin_nontemporal_load(reinterpret_cast<const vec*>(p));
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = t[i];
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = reinterpret_cast<const Elt*>(p)[i];
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (kAligned) {
      typedef Elt vec __attribute__((ext_vector_type(kN)));
      vec t;
#pragma unroll
      for (int i = 0; i < kN; ++i) t[i] = v[i];
      __builtin_nontemporal_store(t, reinterpret_cast<vec*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) reinterpret_cast<Elt*>(p)[i] = v[i];
    }
  }
};

constexpr int kRotaryThreads = 256;

// An item is kP pairs, or, behind them, a run of elements that are copied.
template <int DT, int kP, bool kInterleaved, bool kAligned>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
  constexpr int kB = ChunkElt<DT>::kBytes, kRun = kInterleaved ? 2 * kP : kP, kCopy = kAligned ? kRun : 1;
  constexpr int kAhead = 4;
  typedef RotaryRun<DT, kRun, kAligned> Run;
  const int first = blockIdx.y * a.per_thread, last = min(first + a.per_thread, a.heads);
  uint32_t local, lane;
  a.lanes.divmod(threadIdx.x, local, lane);
  if (local >= a.per_block) return;
  for (uint32_t token = blockIdx.x * a.per_block + local; token < a.tokens; token += gridDim.x * a.per_block)
  for (int at = (int)lane; at < a.items; at += (int)a.lanes.d) {
    uint32_t outer, inner;
    a.inner.divmod(token, outer, inner);
    const uint8_t* x = a.x + (int64_t)outer * a.x_outer + (int64_t)inner * a.x_inner + (int64_t)first * a.x_head;
    uint8_t* y = a.y + (int64_t)outer * a.y_outer + (int64_t)inner * a.y_inner + (int64_t)first * a.y_head;
    if (at >= a.turned) {
      const int64_t off = ((int64_t)2 * a.half + (int64_t)(at - a.turned) * kCopy) * kB;
      for (int h = first; h < last; h += kAhead, x += kAhead * a.x_head, y += kAhead * a.y_head) {
        RotaryRun<DT, kCopy, kAligned> r[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) r[k].load(x + (h + k < last ? k : 0) * a.x_head + off);
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (h + k < last) r[k].store(y + k * a.y_head + off);
      }
      continue;
    }
    float c[kP], s[kP];
    uint32_t skip, row;
    a.position_tokens.divmod(token, skip, row);
#pragma unroll
    for (int i = 0; i < kP; ++i) {
      const int pair = at * kP + i, axis = pair / a.per_axis;
      const int64_t p = (int64_t)row * a.axes + axis;
      const int64_t position = a.wide_positions ? reinterpret_cast<const int64_t*>(a.positions)[p]
                                                : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[p];
      const double t = (double)position * a.turns[pair - axis * a.per_axis];
      const float part = (float)(t - rint(t));
      float sn, cs;
      sincospif(2.f * part, &sn, &cs);
      c[i] = a.amplitude * cs;
      s[i] = a.amplitude * a.sign * sn;
    }
    const int64_t lo = (int64_t)at * kRun * kB, hi = lo + (int64_t)a.half * kB;
    // Heads kAhead at a time, all read before the first is written.
    for (int h = first; h < last; h += kAhead, x += kAhead * a.x_head, y += kAhead * a.y_head) {
      Run p[kAhead], q[kInterleaved ? 1 : kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const uint8_t* xh = x + (h + k < last ? k : 0) * a.x_head;
        p[k].load(xh + lo);
        if constexpr (!kInterleaved) q[k].load(xh + hi);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (h + k >= last) break;
        uint8_t* yh = y + k * a.y_head;
#pragma unroll
        for (int i = 0; i < kP; ++i) {
          auto& eu = kInterleaved ? p[k].v[kInterleaved ? 2 * i : 0] : p[k].v[i];
          auto& ev = kInterleaved ? p[k].v[kInterleaved ? 2 * i + 1 : 0] : q[kInterleaved ? 0 : k].v[i];
          const float u = rotary_value<DT>(eu), v = rotary_value<DT>(ev);
          eu = rotary_round<DT>(u * c[i] - v * s[i]);
          ev = rotary_round<DT>(u * s[i] + v * c[i]);
        }
        p[k].store(yh + lo);
        if constexpr (!kInterleaved) q[k].store(yh + hi);
      }
    }
  }
}

template <int DT, int kP, bool kInterleaved, bool kAligned>
void launch_rotary(RotaryArgs a, int rest, hipStream_t s) {
  constexpr int kCopy = !kAligned ? 1 : kInterleaved ? 2 * kP : kP;
  a.turned = a.half / kP;
  a.items = a.turned + rest / kCopy;
  const int lanes = a.items < kRotaryThreads ? a.items : kRotaryThreads;
  a.lanes = FastDiv((uint32_t)lanes);
  a.per_block = (uint32_t)(kRotaryThreads / lanes);
  // A thread takes several heads only where that leaves threads enough to fill the chip.
  const int64_t want = 1 << 17, threads = (int64_t)a.tokens * lanes;
  int64_t groups = (want + threads - 1) / threads;
  groups = groups > a.heads ? a.heads : groups;
  a.per_thread = (int32_t)((a.heads + groups - 1) / groups);
  const uint32_t need = (a.tokens + a.per_block - 1) / a.per_block, most = 1u << 22;
  const dim3 grid(need < most ? need : most, (unsigned)((a.heads + a.per_thread - 1) / a.per_thread));
  rotary_kernel<DT, kP, kInterleaved, kAligned><<<grid, kRotaryThreads, 0, s>>>(a);
}

template <int DT, bool kInterleaved>
void dispatch_rotary(const RotaryArgs& a, uintptr_t bits, int rest, hipStream_t s) {
  constexpr int kB = ChunkElt<DT>::kBytes;
  // The widest run, up to 16 bytes, that divides the rotated part and the rest and is aligned everywhere.
  auto fits = [&](int p) {
    const int run = kInterleaved ? 2 * p : p;
    return a.half % p == 0 && rest % run == 0 && bits % (uintptr_t)(run * kB) == 0 && (kInterleaved || a.half * kB % (run * kB) == 0);
  };
  if constexpr (kB == 2 && !kInterleaved)
    if (fits(8)) return launch_rotary<DT, 8, kInterleaved, true>(a, rest, s);
  if constexpr (kB == 2 || !kInterleaved)
    if (fits(4)) return launch_rotary<DT, 4, kInterleaved, true>(a, rest, s);
  if (fits(2)) return launch_rotary<DT, 2, kInterleaved, true>(a, rest, s);
  launch_rotary<DT, 1, kInterleaved, false>(a, rest, s);
}

template <int DT>
void rotary_by_layout(const RotaryArgs& a, bool interleaved, uintptr_t bits, int rest, hipStream_t s) {
  if (interleaved) dispatch_rotary<DT, true>(a, bits, rest, s);
  else dispatch_rotary<DT, false>(a, bits, rest, s);
}

// Elements from the first of a tensor to the end of its last.
int64_t rotary_span(int64_t tokens, int64_t inner, int64_t so, int64_t si, int64_t sh, int heads, int head_dim) {
  return (tokens - 1) / inner * so + (tokens < inner ? tokens - 1 : inner - 1) * si + (int64_t)(heads - 1) * sh + head_dim;
}

}  // namespace
}  // namespace terra

using namespace terra;

extern "C" int terra_swin_rotary(const void* x, void* y, const void* positions, const double* turns,
                                 const terra_swin_rotary_desc* d, void* stream) {
  clear_error();
  if (d == nullptr) return fail(TERRA_ERR_NULL, "desc is NULL");
  if (d->dtype != TERRA_DTYPE_F32 && d->dtype != TERRA_DTYPE_BF16 && d->dtype != TERRA_DTYPE_F16)
    return fail(TERRA_ERR_DTYPE, "rotary supports f32, bf16 and f16 (got dtype %d)", d->dtype);
  if (d->position_bits != 32 && d->position_bits != 64)
    return fail(TERRA_ERR_DTYPE, "positions have 32 or 64 bits (got %d)", d->position_bits);
  if (d->tokens < 0 || d->tokens >= (1ll << 31)) return fail(TERRA_ERR_SHAPE, "tokens must be in [0, 2^31) (got %lld)", (long long)d->tokens);
  if (d->heads <= 0 || d->heads > 65535 || d->head_dim <= 0 || d->head_dim > 65536)
    return fail(TERRA_ERR_SHAPE, "1 to 65535 heads of 1 to 65536 (got %d of %d)", d->heads, d->head_dim);
  if (d->dim <= 0 || d->dim > d->head_dim || d->dim % 2 != 0)
    return fail(TERRA_ERR_SHAPE, "dim must be even and in [2, %d] (got %d)", d->head_dim, d->dim);
  if (d->axes <= 0 || d->dim / 2 % d->axes != 0)
    return fail(TERRA_ERR_SHAPE, "the %d pairs are not a whole number for each of %d axes", d->dim / 2, d->axes);
  if (d->inner <= 0 || d->inner >= (1ll << 31) || d->position_tokens <= 0 || d->position_tokens >= (1ll << 31) ||
      d->tokens % d->position_tokens != 0)
    return fail(TERRA_ERR_SHAPE, "inner and position_tokens must be in [1, 2^31), and tokens whole turns of the positions");
  for (int64_t st : {d->x_outer_stride, d->x_inner_stride, d->x_head_stride, d->y_outer_stride, d->y_inner_stride, d->y_head_stride})
    if (st < 0 || st >= (1ll << 40)) return fail(TERRA_ERR_SHAPE, "strides must be in [0, 2^40) (got %lld)", (long long)st);
  if (d->tokens == 0) return TERRA_OK;
  const int elt = dtype_size(d->dtype);
  if (x == nullptr || y == nullptr || positions == nullptr || turns == nullptr)
    return fail(TERRA_ERR_NULL, "x, y, positions or turns is NULL");
  if ((uintptr_t)x % elt != 0 || (uintptr_t)y % elt != 0) return fail(TERRA_ERR_ALIGN, "x or y is not aligned to its elements");
  if ((uintptr_t)positions % (d->position_bits / 8) != 0 || (uintptr_t)turns % 8 != 0)
    return fail(TERRA_ERR_ALIGN, "positions or turns are not aligned");
  // Two elements of y at one place would be written by two threads.
  const int64_t outer_tokens = (d->tokens - 1) / d->inner, inner_tokens = d->tokens < d->inner ? d->tokens : d->inner;
  if ((d->heads > 1 && d->y_head_stride == 0) || (inner_tokens > 1 && d->y_inner_stride == 0) || (outer_tokens > 0 && d->y_outer_stride == 0))
    return fail(TERRA_ERR_SHAPE, "elements of y share a place");
  const bool same = x == y && d->x_outer_stride == d->y_outer_stride && d->x_inner_stride == d->y_inner_stride &&
                    d->x_head_stride == d->y_head_stride;
  const uintptr_t p = (uintptr_t)x, q = (uintptr_t)y;
  const uintptr_t x_bytes = (uintptr_t)(rotary_span(d->tokens, d->inner, d->x_outer_stride, d->x_inner_stride, d->x_head_stride, d->heads, d->head_dim) * elt);
  const uintptr_t y_bytes = (uintptr_t)(rotary_span(d->tokens, d->inner, d->y_outer_stride, d->y_inner_stride, d->y_head_stride, d->heads, d->head_dim) * elt);
  if (!same && p < q + y_bytes && q < p + x_bytes)
    return fail(TERRA_ERR_SHAPE, "y may be x itself, with its strides, and must not overlap it otherwise");
  RotaryArgs a = {};
  a.x = (const uint8_t*)x;
  a.y = (uint8_t*)y;
  a.positions = positions;
  a.turns = turns;
  a.x_outer = d->x_outer_stride * elt, a.x_inner = d->x_inner_stride * elt, a.x_head = d->x_head_stride * elt;
  a.y_outer = d->y_outer_stride * elt, a.y_inner = d->y_inner_stride * elt, a.y_head = d->y_head_stride * elt;
  a.inner = FastDiv((uint32_t)d->inner);
  a.position_tokens = FastDiv((uint32_t)d->position_tokens);
  a.tokens = (uint32_t)d->tokens;
  a.heads = d->heads;
  a.half = d->dim / 2;
  a.axes = d->axes;
  a.per_axis = a.half / d->axes;
  a.wide_positions = d->position_bits == 64;
  a.amplitude = d->amplitude;
  a.sign = d->inverse != 0 ? -1.f : 1.f;
  uintptr_t bits = p | q;
  if (outer_tokens > 0) bits |= (uintptr_t)(a.x_outer | a.y_outer);
  if (inner_tokens > 1) bits |= (uintptr_t)(a.x_inner | a.y_inner);
  if (d->heads > 1) bits |= (uintptr_t)(a.x_head | a.y_head);
  const int rest = same ? 0 : d->head_dim - d->dim;
  hipStream_t s = (hipStream_t)stream;
  if (d->dtype == TERRA_DTYPE_F32) rotary_by_layout<TERRA_DTYPE_F32>(a, d->interleaved != 0, bits, rest, s);
  else if (d->dtype == TERRA_DTYPE_BF16) rotary_by_layout<TERRA_DTYPE_BF16>(a, d->interleaved != 0, bits, rest, s);
  else rotary_by_layout<TERRA_DTYPE_F16>(a, d->interleaved != 0, bits, rest, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TERRA_OK : fail(TERRA_ERR_LAUNCH, "terra_swin_rotary launch failed: %s", hipGetErrorString(e));
}
