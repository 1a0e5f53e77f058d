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
// and cosine serve all of those; its reads are four heads ahead of what it turns.  Bound by memory where
// a token has several heads: 156672 tokens of 16 heads of 128 bf16 228 us, of two heads at a time 240 (a large
// copy moves the same bytes in 250); by the sines and cosines where it has one (200000 of 128: 29 us, 3.5 TB/s; 468750: 65 us, 3.7).
#include "row_chunk.h"

#include <algorithm>
#include <initializer_list>

namespace terra {
namespace {

struct RotaryArgs {
  const uint8_t* x;
  uint8_t* y;
  const void* positions;
  const double* turns;
  int64_t x_outer, x_inner, x_head, y_outer, y_inner, y_head;  // bytes
  FastDiv inner, position_tokens, lanes, per_axis;  // lanes: threads of a token
  uint32_t tokens, per_block;             // tokens of a workgroup
  int32_t turned, items;                  // items of a token that are rotated, and all
  int32_t heads, per_thread;              // heads, of which a thread takes this many
  int32_t half, rest;                     // dim / 2, elements that are copied
  int32_t axes;
  int32_t wide_positions;                 // 64-bit positions
  float amplitude, sign;
};

// kN elements that lie side by side, one access where aligned (to all of them).  kStream: past the
// caches; lines that several accesses share stay there until the last of them.
template <int DT, int kN, bool kAligned, bool kStream>
struct RotaryRun {
  static constexpr int kB = ChunkElt<DT>::kBytes, kWords = (kN * kB + 3) / 4;
  typedef uint32_t Vec __attribute__((ext_vector_type(kWords)));
  uint32_t w[kWords];

  template <typename V>
  static __device__ __forceinline__ V read(const uint8_t* p) {
    if constexpr (kStream) return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
    else return *reinterpret_cast<const V*>(p);
  }
  template <typename V>
  static __device__ __forceinline__ void write(V v, uint8_t* p) {
    if constexpr (kStream) __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
    else *reinterpret_cast<V*>(p) = v;
  }
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (kAligned && kWords == 1) {
      w[0] = read<uint32_t>(p);
    } else if constexpr (kAligned) {
      const Vec v = read<Vec>(p);
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = v[i];
    } else if constexpr (kB == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = (uint32_t)h[2 * i] | (2 * i + 1 < kN ? (uint32_t)h[2 * i + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void store(uint8_t* p) const {
    if constexpr (kAligned && kWords == 1) {
      write(w[0], p);
    } else if constexpr (kAligned) {
      Vec v;
#pragma unroll
      for (int i = 0; i < kWords; ++i) v[i] = w[i];
      write(v, p);
    } else if constexpr (kB == 4) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) reinterpret_cast<uint16_t*>(p)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (DT == TERRA_DTYPE_F32) return __uint_as_float(w[i]);
    const uint32_t v = w[i >> 1];
    if constexpr (DT == TERRA_DTYPE_BF16) return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
    return __half2float(__ushort_as_half((uint16_t)(i & 1 ? v >> 16 : v & 0xffffu)));
  }
  // The run becomes f, rounded once, where `turned` (else it stays).
  __device__ __forceinline__ void turn(const float (&f)[kN], bool turned) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      uint32_t v;
      if constexpr (DT == TERRA_DTYPE_F32) v = __float_as_uint(f[i]);
      else v = pack2<DT>(f[2 * i], 2 * i + 1 < kN ? f[2 * i + 1] : 0.f);
      w[i] = turned ? v : w[i];
    }
  }
};

constexpr int kRotaryThreads = 256;

// An item is kP pairs: of interleaved ones a run of 2 kP elements, else two runs
// of kP.  Behind the rotated items come those that are copied, 2 kP elements each, which go
// through the same loop: a line that holds some of both is read and written at once.  kAhead: heads that a
// thread reads at a time.
template <int DT, int kP, bool kInterleaved, bool kAligned, bool kStream, int kAhead>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
  constexpr int kB = ChunkElt<DT>::kBytes, kRun = kInterleaved ? 2 * kP : kP, kRuns = kInterleaved ? 1 : 2;
  typedef RotaryRun<DT, kRun, kAligned, kStream> Run;
  const int first = blockIdx.y * a.per_thread, last = min(first + a.per_thread, a.heads);
  uint32_t local, lane;
  a.lanes.divmod(threadIdx.x, local, lane);
  if (local >= a.per_block) return;
  for (uint32_t start = blockIdx.x * a.per_block; start < a.tokens; start += gridDim.x * a.per_block) {
    const uint32_t token = start + local;
    if (token >= a.tokens) break;
    uint32_t outer, inner;
    a.inner.divmod(token, outer, inner);
    const uint8_t* x = a.x + (int64_t)outer * a.x_outer + (int64_t)inner * a.x_inner;
    uint8_t* y = a.y + (int64_t)outer * a.y_outer + (int64_t)inner * a.y_inner;
    for (int at = (int)lane; at < a.items; at += (int)a.lanes.d) {
      const bool turned = at < a.turned;
      // Where the item's runs begin in a head; a copied one's second may be past its end (kP = 1).
      const int copied = 2 * a.half + (at - a.turned) * 2 * kP;
      const int lo = (turned ? at * kRun : copied) * kB, hi = (turned ? at * kRun + a.half : copied + kP) * kB;
      const bool both = kAligned || kInterleaved || turned || copied + kP < 2 * a.half + a.rest;
      const bool whole = kAligned || !kInterleaved || turned || copied + 2 * kP <= 2 * a.half + a.rest;
      struct Heads {
        Run r[kAhead][kRuns];
      };
      auto fetch = [&](int h) {
        Heads f;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (h + k >= last) break;
          const uint8_t* xh = x + (int64_t)(h + k) * a.x_head;
          if (whole) {
            f.r[k][0].load(xh + lo);
          } else {  // the last element of an odd rest
            RotaryRun<DT, 1, false, false> one;
            one.load(xh + lo);
            f.r[k][0].w[0] = one.w[0];
          }
          if constexpr (kRuns == 2) f.r[k][1].load(xh + (both ? hi : lo));
        }
        return f;
      };
      Heads ahead = fetch(first);
      float c[kP], s[kP];
      uint32_t skip, row;
      a.position_tokens.divmod(token, skip, row);
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        uint32_t axis = 0, pair = (uint32_t)((turned ? at : 0) * kP + i);
        if (a.axes > 1) a.per_axis.divmod(pair, axis, pair);
        const int64_t p = (int64_t)row * a.axes + axis;
        const int64_t position = a.wide_positions ? reinterpret_cast<const int64_t*>(a.positions)[p]
                                                  : (int64_t)reinterpret_cast<const int32_t*>(a.positions)[p];
        const double t = (double)position * a.turns[pair];
        const float part = (float)(t - rint(t));
        float sn, cs;
        sincospif(2.f * part, &sn, &cs);
        c[i] = a.amplitude * cs;
        s[i] = a.amplitude * a.sign * sn;
      }
      for (int h = first; h < last; h += kAhead) {
        Heads f = ahead;
        if (h + kAhead < last) ahead = fetch(h + kAhead);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          if (h + k >= last) break;
          float u[kRuns][kRun];
#pragma unroll
          for (int i = 0; i < kP; ++i) {
            const float p = f.r[k][0].value(kInterleaved ? 2 * i : i), q = f.r[k][kRuns - 1].value(kInterleaved ? 2 * i + 1 : i);
            u[0][kInterleaved ? 2 * i : i] = p * c[i] - q * s[i];
            u[kRuns - 1][kInterleaved ? 2 * i + 1 : i] = p * s[i] + q * c[i];
          }
#pragma unroll
          for (int i = 0; i < kRuns; ++i) f.r[k][i].turn(u[i], turned);
          uint8_t* yh = y + (int64_t)(h + k) * a.y_head;
          if (whole) {
            f.r[k][0].store(yh + lo);
          } else {
            RotaryRun<DT, 1, false, false> one;
            one.w[0] = f.r[k][0].w[0];
            one.store(yh + lo);
          }
          if constexpr (kRuns == 2)
            if (both) f.r[k][1].store(yh + hi);
        }
      }
    }
  }
}

template <int DT, int kP, bool kInterleaved, bool kAligned>
void launch_rotary(RotaryArgs a, hipStream_t s) {
  a.turned = a.half / kP;
  a.items = a.turned + (a.rest + 2 * kP - 1) / (2 * kP);
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
  // Past the caches where what the lanes of a head read at once is whole lines of 128 bytes (156672 tokens of 16
  // heads of 128 bf16, pairs 64 apart: 231 us, 254 through them; but 312500 of 6 heads of 32, whose lines
  // hold four such pieces: 111 us, 61 through them; 46875 of 16 heads of 80: 100 and 59).
  constexpr int kB = ChunkElt<DT>::kBytes;
  const bool lines = kInterleaved ? (2 * a.half + a.rest) * kB % 128 == 0 : a.half * kB % 128 == 0 && a.rest * kB % 256 == 0;
  // Four heads ahead take registers that a thread of few heads has better use for (200000 x 1 of 128: 29 us, 36 so).
  const bool many = a.per_thread >= 4;
  if constexpr (kAligned)
    if (lines) {
      if (many) rotary_kernel<DT, kP, kInterleaved, true, true, 4><<<grid, kRotaryThreads, 0, s>>>(a);
      else rotary_kernel<DT, kP, kInterleaved, true, true, 1><<<grid, kRotaryThreads, 0, s>>>(a);
      return;
    }
  if (many) rotary_kernel<DT, kP, kInterleaved, kAligned, false, 4><<<grid, kRotaryThreads, 0, s>>>(a);
  else rotary_kernel<DT, kP, kInterleaved, kAligned, false, 1><<<grid, kRotaryThreads, 0, s>>>(a);
}

template <int DT, bool kInterleaved>
void dispatch_rotary(const RotaryArgs& a, uintptr_t bits, hipStream_t s) {
  constexpr int kB = ChunkElt<DT>::kBytes;
  // The widest run, of 16 bytes down to 4, that divides the rotated part and the rest and is aligned everywhere.
  auto fits = [&](int p) {
    const int run = kInterleaved ? 2 * p : p;
    return a.half % p == 0 && a.rest % (2 * p) == 0 && bits % (uintptr_t)(run * kB) == 0;
  };
  if constexpr (kB == 2 && !kInterleaved)
    if (fits(8)) return launch_rotary<DT, 8, kInterleaved, true>(a, s);
  if constexpr (kB == 2 || !kInterleaved)
    if (fits(4)) return launch_rotary<DT, 4, kInterleaved, true>(a, s);
  if (fits(2)) return launch_rotary<DT, 2, kInterleaved, true>(a, s);
  launch_rotary<DT, 1, kInterleaved, false>(a, s);
}

template <int DT>
void rotary_by_layout(const RotaryArgs& a, bool interleaved, uintptr_t bits, hipStream_t s) {
  if (interleaved) dispatch_rotary<DT, true>(a, bits, s);
  else dispatch_rotary<DT, false>(a, bits, s);
}

// Elements from the first of a tensor to the end of its last.
int64_t rotary_span(int64_t tokens, int64_t inner, int64_t so, int64_t si, int64_t sh, int heads, int head_dim) {
  return (tokens - 1) / inner * so + (tokens < inner ? tokens - 1 : inner - 1) * si + (int64_t)(heads - 1) * sh + head_dim;
}

struct Level {
  int64_t stride, size;
};

// Whether each level of a tensor steps over all that the finer ones reach, so that no two elements share a place.
bool strides_nest(const Level (&levels)[4]) {
  Level by_stride[4];
  int count = 0;
  for (const Level& l : levels)
    if (l.size > 1) by_stride[count++] = l;
  std::sort(by_stride, by_stride + count, [](const Level& a, const Level& b) { return a.stride < b.stride; });
  __int128 reach = 1;
  for (int i = 0; i < count; ++i) {
    if (by_stride[i].stride < reach) return false;
    reach += (__int128)(by_stride[i].size - 1) * by_stride[i].stride;
  }
  return true;
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
  if (!strides_nest({{1, d->head_dim}, {d->y_head_stride, d->heads}, {d->y_inner_stride, inner_tokens}, {d->y_outer_stride, outer_tokens + 1}}))
    return fail(TERRA_ERR_SHAPE, "y's strides do not nest: elements of it may share a place");
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
  a.per_axis = FastDiv((uint32_t)(a.half / d->axes));
  a.wide_positions = d->position_bits == 64;
  a.amplitude = d->amplitude;
  a.sign = d->inverse != 0 ? -1.f : 1.f;
  uintptr_t bits = p | q;
  if (outer_tokens > 0) bits |= (uintptr_t)(a.x_outer | a.y_outer);
  if (inner_tokens > 1) bits |= (uintptr_t)(a.x_inner | a.y_inner);
  if (d->heads > 1) bits |= (uintptr_t)(a.x_head | a.y_head);
  a.rest = same ? 0 : d->head_dim - d->dim;
  hipStream_t s = (hipStream_t)stream;
  if (d->dtype == TERRA_DTYPE_F32) rotary_by_layout<TERRA_DTYPE_F32>(a, d->interleaved != 0, bits, s);
  else if (d->dtype == TERRA_DTYPE_BF16) rotary_by_layout<TERRA_DTYPE_BF16>(a, d->interleaved != 0, bits, s);
  else rotary_by_layout<TERRA_DTYPE_F16>(a, d->interleaved != 0, bits, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TERRA_OK : fail(TERRA_ERR_LAUNCH, "terra_swin_rotary launch failed: %s", hipGetErrorString(e));
}
