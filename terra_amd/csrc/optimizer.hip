// The update of the parameters: the norm of all gradients as one vector, and
// an AdamW step over many tensors at once, its moments in 32 bits or in 8
// (the formulas stand at the entry points' declarations).
//
// The tensors of a launch are listed in its arguments, up to kListed of them,
// so nothing has to be copied to the device before it and a captured graph
// keeps them; a workgroup has a chunk of one tensor, found by a binary search.
// All are bound by memory.  151 million elements (12 blocks of 1024 channels): the norm of bf16 gradients 55 us, 5.4 TB/s, by
// 16-byte loads, eight ahead (by 4-byte ones 110); a clipped fp32 step 873 us, 5.5 TB/s, with moments in 8 bits
// 557 us, 5.4 TB/s (a large copy moves 5.35).  Small sets are a launch each: 17 tensors of one block of 96 channels 9 us.
#include "row_chunk.h"

#include <algorithm>
#include <exception>
#include <initializer_list>
#include <vector>

namespace terra {
namespace {

constexpr int kListed = 64;  // tensors of a launch: 56 bytes each, of 4 KB of arguments

// Of the tensors whose chunks begin at start[0] <= start[1] <= ..., the one that holds `chunk`.
__device__ __forceinline__ int tensor_of(const uint32_t* start, int count, uint32_t chunk) {
  int lo = 0, hi = count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (start[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int DT>
__device__ __forceinline__ float one_value(const uint8_t* p, int64_t i) {
  if constexpr (DT == TERRA_DTYPE_F32) return reinterpret_cast<const float*>(p)[i];
  const uint16_t v = reinterpret_cast<const uint16_t*>(p)[i];
  if constexpr (DT == TERRA_DTYPE_BF16) return bf16_bits_to_f32(v);
  return __half2float(__ushort_as_half(v));
}

// Elements i .. i + 3, of which the first n are there (0 in the others); kVec: all of
// them, aligned to four elements.
template <int DT, bool kVec>
__device__ __forceinline__ void four_values(const uint8_t* p, int64_t i, int n, float (&f)[4]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < n ? one_value<DT>(p, i + j) : 0.f;
  } else if constexpr (DT == TERRA_DTYPE_F32) {
    const stream_u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const stream_u32x4*>(p + i * 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(v[j]);
  } else {
    const stream_u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const stream_u32x2*>(p + i * 2));
    RowChunk<DT> r;
    r.q[0][0] = v[0];
    r.q[0][1] = v[1];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = chunk_value<DT>(r, j);
  }
}

template <int DT, bool kVec>
__device__ __forceinline__ void put_four(uint8_t* p, int64_t i, int n, const float (&f)[4]) {
  if constexpr (!kVec) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) {
        if constexpr (DT == TERRA_DTYPE_F32) reinterpret_cast<float*>(p)[i + j] = f[j];
        else reinterpret_cast<uint16_t*>(p)[i + j] = (uint16_t)pack2<DT>(f[j], 0.f);
      }
  } else if constexpr (DT == TERRA_DTYPE_F32) {
    const stream_u32x4 v = {__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    __builtin_nontemporal_store(v, reinterpret_cast<stream_u32x4*>(p + i * 4));
  } else {
    const stream_u32x2 v = {pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3])};
    __builtin_nontemporal_store(v, reinterpret_cast<stream_u32x2*>(p + i * 2));
  }
}

// ---- the norm of the gradients --------------------------------------------------

constexpr int kNormThreads = 256;
constexpr int64_t kNormChunk = 16384;  // elements of a workgroup

constexpr int kGradListed = 160;  // gradients of a launch: 21 bytes each

struct GradList {
  const uint8_t* data[kGradListed];
  int64_t numel[kGradListed];
  uint32_t start[kGradListed];
  uint8_t dtype[kGradListed];
  double* partials;
  int32_t count;
};
static_assert(sizeof(GradList) <= 4096, "arguments of a launch");

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
  return v;
}

// The thread's sum of squares of elements begin .. end - 1 (begin a multiple of kNormChunk).  Loads of
// 16 bytes, kNormAhead of them before the first is used.
constexpr int kNormAhead = 8;

template <int DT>
__device__ __forceinline__ double squares(const uint8_t* g, int64_t begin, int64_t end) {
  constexpr int kB = ChunkElt<DT>::kBytes, kN = 16 / kB;
  double sum[2] = {0.0, 0.0};
  int64_t i = begin + threadIdx.x * kN;
  if ((uintptr_t)g % 16 == 0) {
    for (; i + (kNormAhead - 1) * kNormThreads * kN + kN <= end; i += kNormAhead * kNormThreads * kN) {
      stream_u32x4 v[kNormAhead];
#pragma unroll
      for (int u = 0; u < kNormAhead; ++u)
        v[u] = __builtin_nontemporal_load(reinterpret_cast<const stream_u32x4*>(g + (i + u * kNormThreads * kN) * kB));
#pragma unroll
      for (int u = 0; u < kNormAhead; ++u) {
        RowChunk<DT> r;
        r.q[0] = v[u];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const double f = (double)chunk_value<DT>(r, j);
          sum[j & 1] = fma(f, f, sum[j & 1]);
        }
      }
    }
    for (; i + kN <= end; i += kNormThreads * kN) {
      RowChunk<DT> r;
      r.q[0] = *reinterpret_cast<const stream_u32x4*>(g + i * kB);
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const double f = (double)chunk_value<DT>(r, j);
        sum[j & 1] = fma(f, f, sum[j & 1]);
      }
    }
  }
  for (; i < end; i += kNormThreads * kN)
#pragma unroll
    for (int j = 0; j < kN; ++j)
      if (i + j < end) {
        const double f = (double)one_value<DT>(g, i + j);
        sum[j & 1] = fma(f, f, sum[j & 1]);
      }
  return sum[0] + sum[1];
}

__global__ __launch_bounds__(kNormThreads) void gradient_norm_kernel(const GradList a) {
  __shared__ double s[kNormThreads / 64];
  const int t = tensor_of(a.start, a.count, blockIdx.x);
  const uint8_t* g = a.data[t];
  const int64_t begin = (int64_t)(blockIdx.x - a.start[t]) * kNormChunk;
  const int64_t end = begin + kNormChunk < a.numel[t] ? begin + kNormChunk : a.numel[t];
  const int dtype = a.dtype[t];
  double sum = dtype == TERRA_DTYPE_F32    ? squares<TERRA_DTYPE_F32>(g, begin, end)
               : dtype == TERRA_DTYPE_BF16 ? squares<TERRA_DTYPE_BF16>(g, begin, end)
                                           : squares<TERRA_DTYPE_F16>(g, begin, end);
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.partials[blockIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
}

constexpr int kResultThreads = 1024;

__global__ __launch_bounds__(kResultThreads) void gradient_norm_result_kernel(const double* partials, int64_t count,
                                                                              double max_norm, float* result) {
  __shared__ double s[kResultThreads / 64];
  double sum = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kResultThreads) sum += partials[i];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  sum = 0.0;
  for (int w = 0; w < kResultThreads / 64; ++w) sum += s[w];
  const double norm = sqrt(sum), factor = max_norm / (norm + 1e-6);
  const float shown = (float)norm;
  result[0] = shown;
  result[1] = max_norm > 0.0 ? (factor > 1.0 ? 1.f : (float)factor) : 1.f;  // NaN for a NaN norm
  result[2] = fabsf(shown) <= 3.4028235e38f ? 0.f : 1.f;
}

// ---- AdamW ----------------------------------------------------------------------

constexpr int kAdamThreads = 256;
// Elements of a workgroup: fewer in a set that would not fill the chip (110000 elements 4.8 us, 6.2 with the larger
// chunks, with moments in 8 bits 5.8 and 9.7; 4 million 19.2, 20.5 and 16.6, 17.3; 64 million the same or worse).
constexpr uint32_t kAdamChunk = 8192, kAdamSmallChunk = 2048;
constexpr int64_t kAdamSmallSet = 1 << 22;
constexpr int kScaled = 256;          // elements that share a scale

struct AdamEntry {
  uint8_t* param;
  const uint8_t* grad;
  uint8_t* first;
  uint8_t* second;
  float* scales;
  int64_t numel;
};

struct AdamList {
  AdamEntry tensor[kListed];
  uint32_t start[kListed];
  uint32_t index[kListed];
  int32_t count;
  int32_t maximize;
  uint32_t chunk;
  double lr, beta1, beta2, eps, decay;
  int64_t step;
  const int64_t* step_ptr;
  const float *lr_ptr, *grad_factor, *found_inf;
  const uint64_t* seed;
  uint32_t stream;
};
static_assert(sizeof(AdamList) <= 4096, "arguments of a launch");

// beta^n by repeated squaring, in 64 bits.
__device__ __forceinline__ double power(double beta, int64_t n) {
  double r = 1.0;
  for (; n > 0; n >>= 1, beta *= beta)
    if (n & 1) r *= beta;
  return r;
}

// What a step multiplies by, the same for all elements.
struct AdamStep {
  float keep, rate, root, eps;  // 1 - lr decay, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), eps
  float factor;                 // of the gradients
  uint32_t step;

  __device__ __forceinline__ explicit AdamStep(const AdamList& a) {
    const int64_t t = a.step_ptr != nullptr ? *a.step_ptr : a.step;
    const double lr = a.lr_ptr != nullptr ? (double)*a.lr_ptr : a.lr;
    keep = (float)(1.0 - lr * a.decay);
    rate = (float)(lr / (1.0 - power(a.beta1, t)));
    root = (float)(1.0 / sqrt(1.0 - power(a.beta2, t)));
    eps = (float)a.eps;
    factor = a.grad_factor != nullptr ? *a.grad_factor : 1.f;
    if (a.maximize) factor = -factor;
    step = (uint32_t)t;
  }
  // r: the second moment's root.  The quotient by the hardware's reciprocal, an ulp: what a step takes off is off by that.
  __device__ __forceinline__ float updated(float p, float m, float r) const {
    return fmaf(-rate * m, __builtin_amdgcn_rcpf(fmaf(r, root, eps)), p * keep);
  }
};

// Four elements of a lane.
template <int DTP, int DTG, bool kVec>
struct AdamElements {
  float p[4], g[4], m[4], v[4];

  __device__ __forceinline__ void load(const AdamEntry& e, int64_t i, int n) {
    four_values<DTP, kVec>(e.param, i, n, p);
    four_values<DTG, kVec>(e.grad, i, n, g);
    four_values<TERRA_DTYPE_F32, kVec>(e.first, i, n, m);
    four_values<TERRA_DTYPE_F32, kVec>(e.second, i, n, v);
  }
  __device__ __forceinline__ void step(const AdamStep& st, float b1, float c1, float b2, float c2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float d = g[j] * st.factor;
      m[j] = fmaf(c1, d, b1 * m[j]);
      v[j] = fmaf(c2 * d, d, b2 * v[j]);
      p[j] = st.updated(p[j], m[j], sqrtf(v[j]));
    }
  }
  __device__ __forceinline__ void store(const AdamEntry& e, int64_t i, int n) const {
    put_four<DTP, kVec>(e.param, i, n, p);
    put_four<TERRA_DTYPE_F32, kVec>(e.first, i, n, m);
    put_four<TERRA_DTYPE_F32, kVec>(e.second, i, n, v);
  }
};

constexpr int kAdamAhead = 2;  // groups of four that a thread reads before it writes the first

template <int DTP, int DTG>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(const AdamList a) {
  if (a.found_inf != nullptr && *a.found_inf != 0.f) return;
  const int t = tensor_of(a.start, a.count, blockIdx.x);
  const AdamEntry e = a.tensor[t];
  const AdamStep st(a);
  const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2);
  const int64_t begin = (int64_t)(blockIdx.x - a.start[t]) * a.chunk;
  const int64_t end = begin + a.chunk < e.numel ? begin + a.chunk : e.numel;
  const bool vec = (uintptr_t)e.param % (4 * ChunkElt<DTP>::kBytes) == 0 && (uintptr_t)e.grad % (4 * ChunkElt<DTG>::kBytes) == 0 &&
                   ((uintptr_t)e.first | (uintptr_t)e.second) % 16 == 0;
  constexpr int kStride = kAdamThreads * 4;
  int64_t i = begin + threadIdx.x * 4;
  if (vec)
    for (; i + (kAdamAhead - 1) * kStride + 4 <= end; i += kAdamAhead * kStride) {
      AdamElements<DTP, DTG, true> q[kAdamAhead];
#pragma unroll
      for (int u = 0; u < kAdamAhead; ++u) q[u].load(e, i + u * kStride, 4);
#pragma unroll
      for (int u = 0; u < kAdamAhead; ++u) {
        q[u].step(st, b1, c1, b2, c2);
        q[u].store(e, i + u * kStride, 4);
      }
    }
  for (; i < end; i += kStride) {
    const int n = (int)(end - i < 4 ? end - i : 4);
    AdamElements<DTP, DTG, false> q;
    q.load(e, i, n);
    q.step(st, b1, c1, b2, c2);
    q.store(e, i, n);
  }
}

// ---- moments in 8 bits ----------------------------------------------------------
// The moments in 64 bits: the first one's terms may cancel, the second's squares
// leave the range of 32 (gradients below 10^-19).  From there on in 32 bits.

// The largest of a 32-bit number over the wave's lanes (every lane ends with it).
__device__ __forceinline__ uint32_t wave_largest(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false));   // lane ^ 1
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, false));   // lane ^ 2
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));  // the other quad of eight
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, false));  // the other eight of a row
  auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(p[0], p[1]);
  p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(p[0], p[1]);
}

// Four e4m3 codes of values of at most 448 in size.
__device__ __forceinline__ uint32_t fp8_codes(const float (&f)[4]) {
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
}
template <int kJ>
__device__ __forceinline__ float fp8_value(uint32_t codes) { return __builtin_amdgcn_cvt_f32_fp8((int)codes, kJ); }

constexpr float kLargestCode = 448.f, kSmallestCode = 0.001953125f;

// A value on one of the two codes next to r >= 0 (at most 448 and a rounding): of low <= r < high the
// upper one where r^2 - low^2 > u (high^2 - low^2).  Squares of codes are exact.  Without branches: a code's
// step is 2^-3 of the power of two below r, from 2^-6 down 2^-9.
__device__ __forceinline__ float root_code(float r, uint32_t draw) {
  const float c = fminf(r, kLargestCode);
  const uint32_t power = max(__float_as_uint(c), 0x3c800000u) & 0x7f800000u;  // of two, at least 2^-6
  const float step = __uint_as_float(power - (3u << 23)), per_step = __uint_as_float((257u << 23) - power);
  const float low = floorf(c * per_step) * step, high = low + step;
  const float l2 = low * low, span = fmaf(high, high, -l2);
  const float u = fmaf((float)draw, 1.f / 65536.f, 0.5f / 65536.f);
  const float v = fmaf(c, c, -l2) > u * span ? high : low;
  const float held = __builtin_amdgcn_fmed3f(v, kSmallestCode, kLargestCode);
  return r > 0.f ? held : 0.f;
}

__device__ __forceinline__ ChunkDraws adam_draws(uint64_t seed, uint32_t chunk, uint32_t tensor, uint32_t step, uint32_t stream) {
  uint32_t c0 = chunk, c1 = tensor, c2 = step, c3 = stream;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)b;
    c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// The value of lane `from` (the same in all lanes) of a 64-bit number.
__device__ __forceinline__ double lane_value(double v, int from) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, from), hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), from);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

// Four elements of a lane.
struct AdamFour {
  float p[4], g[4];
  uint32_t first, second;  // codes

  template <int DTP, int DTG>
  __device__ __forceinline__ void load(const AdamEntry& e, int64_t i, int n, bool whole) {
    if (whole) {
      four_values<DTP, true>(e.param, i, 4, p);
      four_values<DTG, true>(e.grad, i, 4, g);
      first = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(e.first + i));
      second = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(e.second + i));
    } else {
      four_values<DTP, false>(e.param, i, n, p);
      four_values<DTG, false>(e.grad, i, n, g);
      first = second = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        first |= j < n ? (uint32_t)e.first[i + j] << (8 * j) : 0u;
        second |= j < n ? (uint32_t)e.second[i + j] << (8 * j) : 0u;
      }
    }
  }
  template <int DTP>
  __device__ __forceinline__ void store(const AdamEntry& e, int64_t i, int n, bool whole) const {
    if (whole) {
      put_four<DTP, true>(e.param, i, 4, p);
      __builtin_nontemporal_store(first, reinterpret_cast<uint32_t*>(e.first + i));
      __builtin_nontemporal_store(second, reinterpret_cast<uint32_t*>(e.second + i));
    } else {
      put_four<DTP, false>(e.param, i, n, p);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) {
          e.first[i + j] = (uint8_t)(first >> (8 * j));
          e.second[i + j] = (uint8_t)(second >> (8 * j));
        }
    }
  }
};

// A wave takes two blocks of 256 elements at a time, four of each a lane: neighbouring lanes
// then hold the halves of two chunks of eight and share their draws, as in half_draws.
template <int DTP, int DTG>
__global__ __launch_bounds__(kAdamThreads) void adamw_8bit_kernel(const AdamList a) {
  if (a.found_inf != nullptr && *a.found_inf != 0.f) return;
  const int t = tensor_of(a.start, a.count, blockIdx.x);
  const AdamEntry e = a.tensor[t];
  const AdamStep st(a);
  const uint64_t seed = *a.seed;
  const double c1 = (1.0 - a.beta1) * (double)st.factor, c2 = (1.0 - a.beta2) * (double)st.factor * (double)st.factor;
  const int64_t blocks = (e.numel + kScaled - 1) / kScaled;
  const uint32_t most = a.chunk / kScaled;
  const int64_t begin = (int64_t)(blockIdx.x - a.start[t]) * most;
  const int64_t end = begin + most < blocks ? begin + most : blocks;
  const int lane = threadIdx.x & 63;
  const bool vec = (uintptr_t)e.param % (4 * ChunkElt<DTP>::kBytes) == 0 && (uintptr_t)e.grad % (4 * ChunkElt<DTG>::kBytes) == 0 &&
                   ((uintptr_t)e.first | (uintptr_t)e.second) % 4 == 0;
  for (int64_t b = begin + 2 * (threadIdx.x >> 6); b < end; b += 2 * (kAdamThreads / 64)) {
    AdamFour q[2];
    int n[2];
    double scale_m[2], scale_r[2];
    const bool whole = vec && (b + 2) * kScaled <= e.numel;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t i = (b + k) * kScaled + lane * 4, left = e.numel - i;
      n[k] = left >= 4 ? 4 : left > 0 ? (int)left : 0;
      q[k].template load<DTP, DTG>(e, i, n[k], whole);
      const bool there = b + k < end;
      scale_m[k] = there ? (double)e.scales[b + k] : 0.0;
      scale_r[k] = there ? (double)e.scales[blocks + b + k] : 0.0;
    }
    double m[2][4];
    float r[2][4];
    uint32_t big_m[2], big_r[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float fm[4] = {fp8_value<0>(q[k].first), fp8_value<1>(q[k].first), fp8_value<2>(q[k].first), fp8_value<3>(q[k].first)};
      const float fr[4] = {fp8_value<0>(q[k].second), fp8_value<1>(q[k].second), fp8_value<2>(q[k].second), fp8_value<3>(q[k].second)};
      const double dm = a.beta1 * scale_m[k], dv = a.beta2 * scale_r[k] * scale_r[k];
      double v[4];
      uint32_t away = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const double g = (double)q[k].g[j];
        m[k][j] = fma((double)fm[j], dm, c1 * g);
        v[j] = fma((double)(fr[j] * fr[j]), dv, c2 * g * g);
        // How far the exponent is above 2^-100 (below it, and for 0, a large number).
        away = max(away, (uint32_t)((uint64_t)__double_as_longlong(v[j]) >> 32) - ((1023u - 100u) << 20));
        r[k][j] = __builtin_amdgcn_sqrtf((float)v[j]);
      }
      if (__builtin_amdgcn_ballot_w64(away > (220u << 20)) != 0)  // not all in 2^-100 .. 2^120
#pragma unroll
        for (int j = 0; j < 4; ++j) r[k][j] = (float)sqrt(v[j]);
      big_m[k] = big_r[k] = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float m32 = (float)m[k][j];
        q[k].p[j] = st.updated(q[k].p[j], m32, r[k][j]);
        big_m[k] = max(big_m[k], __float_as_uint(m32) & 0x7fffffffu);  // NaN above infinity above the others
        big_r[k] = max(big_r[k], __float_as_uint(r[k][j]) & 0x7fffffffu);
      }
      big_m[k] = wave_largest(big_m[k]);
      big_r[k] = wave_largest(big_r[k]);
    }
    // The scales, and their reciprocals: each of the four in the lanes of its number.  With an infinity or a NaN the scale is
    // infinite, and all of the block NaN when it is read again.
    const uint32_t big = lane & 2 ? (lane & 1 ? big_r[1] : big_m[1]) : (lane & 1 ? big_r[0] : big_m[0]);
    const float scale = big >= 0x7f800000u ? __builtin_inff() : __uint_as_float(big) / kLargestCode;
    const double inverse = scale > 0.f ? 1.0 / (double)scale : 0.0;
    // The even lane's draws are of the first block's chunk, the odd one's of the second's.
    const uint32_t pair = (uint32_t)(b * (kScaled / 8)) + (uint32_t)(lane >> 1);
    const ChunkDraws d = adam_draws(seed, pair + (lane & 1) * (kScaled / 8), a.index[t], st.step, a.stream);
    const uint32_t other0 = lane_xor1(lane & 1 ? d.w[0] : d.w[2]), other1 = lane_xor1(lane & 1 ? d.w[1] : d.w[3]);
    const uint32_t w[2][2] = {{lane & 1 ? other0 : d.w[0], lane & 1 ? other1 : d.w[1]}, {lane & 1 ? d.w[2] : other0, lane & 1 ? d.w[3] : other1}};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const double inv_m = lane_value(inverse, 2 * k), inv_r = lane_value(inverse, 2 * k + 1);
      float y[4], z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y[j] = __builtin_amdgcn_fmed3f((float)(m[k][j] * inv_m), -kLargestCode, kLargestCode);
        const float part = (float)((double)r[k][j] * inv_r);
        z[j] = root_code(part, j & 1 ? w[k][j >> 1] >> 16 : w[k][j >> 1] & 0xffffu);
      }
      q[k].first = fp8_codes(y);
      q[k].second = fp8_codes(z);
      q[k].template store<DTP>(e, (b + k) * kScaled + lane * 4, n[k], whole);
    }
    if (lane < 4 && b + (lane >> 1) < end) e.scales[(lane & 1 ? blocks : 0) + b + (lane >> 1)] = scale;
  }
}

}  // namespace

// ---- entry points ---------------------------------------------------------------

namespace {

constexpr int64_t kMostElements = 1ll << 35;   // of a tensor: an element's chunk of eight has 32 bits in the counter
constexpr uint32_t kMostChunks = 1u << 22;     // workgroups of a launch

bool float_dtype(int d) { return d == TERRA_DTYPE_F32 || d == TERRA_DTYPE_BF16 || d == TERRA_DTYPE_F16; }

int optimizer_launched(const char* what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? TERRA_OK : fail(TERRA_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

int grad_counts(const terra_swin_tensor* grads, int count, int64_t* partials) {
  if (count < 0) return fail(TERRA_ERR_SHAPE, "count must be >= 0");
  if (count > 0 && grads == nullptr) return fail(TERRA_ERR_NULL, "grads is NULL");
  *partials = 0;
  for (int i = 0; i < count; ++i) {
    const int64_t n = grads[i].numel;
    if (!float_dtype(grads[i].dtype)) return fail(TERRA_ERR_DTYPE, "gradients are f32, bf16 or f16 (%d is %d)", i, grads[i].dtype);
    if (n < 0 || n >= kMostElements) return fail(TERRA_ERR_SHAPE, "gradient %d has %lld elements: at most 2^35 - 1", i, (long long)n);
    *partials += (n + kNormChunk - 1) / kNormChunk;
  }
  if (*partials >= (1ll << 31)) return fail(TERRA_ERR_SHAPE, "the gradients have too many elements");
  return TERRA_OK;
}

struct Span {
  uintptr_t begin, end;
  bool written;
};

// Whether a range that is written meets another one: sorted by their beginnings,
// each is compared with the furthest end before it.
bool spans_meet(std::vector<Span>& spans) {
  std::sort(spans.begin(), spans.end(), [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;  // the furthest ends so far
  for (const Span& s : spans) {
    if (s.begin < written || (s.written && s.begin < any)) return true;
    any = std::max(any, s.end);
    if (s.written) written = std::max(written, s.end);
  }
  return false;
}

// The pair of types of a tensor, and whether its moments are in 8 bits, as one number.
int adamw_kind(const terra_swin_adamw_tensor& t) {
  constexpr int F = TERRA_DTYPE_F32, B = TERRA_DTYPE_BF16;
  const int p = t.param_dtype, g = t.grad_dtype;
  const int pair = p == F ? (g == F ? 0 : g == B ? 1 : 2) : p == B ? (g == B ? 3 : 4) : (g == F ? 6 : 5);
  return 2 * pair + (t.scales != nullptr ? 1 : 0);
}

template <int DTP, int DTG>
void launch_adamw(bool scaled, const AdamList& a, uint32_t chunks, hipStream_t s) {
  if (scaled) adamw_8bit_kernel<DTP, DTG><<<chunks, kAdamThreads, 0, s>>>(a);
  else adamw_kernel<DTP, DTG><<<chunks, kAdamThreads, 0, s>>>(a);
}

void dispatch_adamw(int kind, const AdamList& a, uint32_t chunks, hipStream_t s) {
  constexpr int F = TERRA_DTYPE_F32, B = TERRA_DTYPE_BF16, H = TERRA_DTYPE_F16;
  const bool scaled = kind & 1;
  switch (kind >> 1) {
    case 0: return launch_adamw<F, F>(scaled, a, chunks, s);
    case 1: return launch_adamw<F, B>(scaled, a, chunks, s);
    case 2: return launch_adamw<F, H>(scaled, a, chunks, s);
    case 3: return launch_adamw<B, B>(scaled, a, chunks, s);
    case 4: return launch_adamw<B, F>(scaled, a, chunks, s);
    case 5: return launch_adamw<H, H>(scaled, a, chunks, s);
    default: return launch_adamw<H, F>(scaled, a, chunks, s);
  }
}

int adamw_checked(const terra_swin_adamw_tensor* tensors, int count, const terra_swin_adamw_desc* d, hipStream_t stream) {
  if (d == nullptr) return fail(TERRA_ERR_NULL, "desc is NULL");
  if (count < 0) return fail(TERRA_ERR_SHAPE, "count must be >= 0");
  if (count > 0 && tensors == nullptr) return fail(TERRA_ERR_NULL, "tensors is NULL");
  for (double beta : {d->beta1, d->beta2})
    if (!(beta >= 0.0 && beta < 1.0)) return fail(TERRA_ERR_SHAPE, "betas must be in [0, 1) (got %g)", beta);
  if (!(d->eps >= 0.0) || !(d->weight_decay >= 0.0) || (d->lr_ptr == nullptr && !(d->lr >= 0.0)))
    return fail(TERRA_ERR_SHAPE, "lr, eps and weight_decay must be >= 0 (got %g, %g, %g)", d->lr, d->eps, d->weight_decay);
  if (d->step_ptr == nullptr && d->step < 1) return fail(TERRA_ERR_SHAPE, "step counts from 1 (got %lld)", (long long)d->step);
  if (((uintptr_t)d->step_ptr | (uintptr_t)d->seed) % 8 != 0 ||
      ((uintptr_t)d->lr_ptr | (uintptr_t)d->grad_factor | (uintptr_t)d->found_inf) % 4 != 0)
    return fail(TERRA_ERR_ALIGN, "step, seed, lr, grad_factor or found_inf is not aligned");
  std::vector<Span> spans;
  spans.reserve((size_t)count * 5);
  uint32_t kinds = 0;  // the pairs of types, by kind of moments, that the list holds
  int64_t total = 0;
  for (int i = 0; i < count; ++i) {
    const terra_swin_adamw_tensor& t = tensors[i];
    const int pd = t.param_dtype, gd = t.grad_dtype;
    if (!float_dtype(pd) || !float_dtype(gd) || (pd != gd && pd != TERRA_DTYPE_F32 && gd != TERRA_DTYPE_F32))
      return fail(TERRA_ERR_DTYPE, "parameters and gradients are f32, bf16 or f16, of one dtype unless one is f32 (%d: %d and %d)", i, pd, gd);
    if (t.numel < 0 || t.numel >= kMostElements)
      return fail(TERRA_ERR_SHAPE, "tensor %d has %lld elements: at most 2^35 - 1", i, (long long)t.numel);
    const bool scaled = t.scales != nullptr;
    if (scaled && d->seed == nullptr) return fail(TERRA_ERR_NULL, "moments in 8 bits need a seed");
    if (t.numel == 0) continue;
    kinds |= 1u << adamw_kind(t);
    total = total < kAdamSmallSet ? total + t.numel : total;
    const uintptr_t pe = dtype_size(pd), ge = dtype_size(gd), me = scaled ? 1 : 4;
    const uintptr_t p = (uintptr_t)t.param, g = (uintptr_t)t.grad, m = (uintptr_t)t.exp_avg, v = (uintptr_t)t.exp_avg_sq, n = (uintptr_t)t.numel;
    if (!p || !g || !m || !v) return fail(TERRA_ERR_NULL, "tensor %d: the parameter, its gradient or a moment is NULL", i);
    if (p % pe != 0 || g % ge != 0 || (m | v) % me != 0 || (uintptr_t)t.scales % 4 != 0)
      return fail(TERRA_ERR_ALIGN, "tensor %d is not aligned to its elements", i);
    spans.push_back({p, p + n * pe, true});
    spans.push_back({g, g + n * ge, false});
    spans.push_back({m, m + n * me, true});
    spans.push_back({v, v + n * me, true});
    if (scaled) spans.push_back({(uintptr_t)t.scales, (uintptr_t)t.scales + (n + kScaled - 1) / kScaled * 8, true});
  }
  if (spans_meet(spans)) return fail(TERRA_ERR_SHAPE, "parameters, moments and scales must not overlap each other or the gradients");
  if (kinds == 0) return TERRA_OK;
  AdamList a = {};
  a.maximize = d->maximize;
  a.chunk = total < kAdamSmallSet ? kAdamSmallChunk : kAdamChunk;
  a.lr = d->lr, a.beta1 = d->beta1, a.beta2 = d->beta2, a.eps = d->eps, a.decay = d->weight_decay;
  a.step = d->step;
  a.step_ptr = (const int64_t*)d->step_ptr;
  a.lr_ptr = d->lr_ptr, a.grad_factor = d->grad_factor, a.found_inf = d->found_inf;
  a.seed = (const uint64_t*)d->seed;
  a.stream = d->stream_id;
  for (int kind = 0; kinds >> kind != 0; ++kind) {
    if ((kinds >> kind & 1u) == 0) continue;
    uint32_t chunks = 0;
    auto launch = [&] {
      if (a.count > 0) dispatch_adamw(kind, a, chunks, stream);
      a.count = 0;
      chunks = 0;
    };
    for (int i = 0; i < count; ++i) {
      const terra_swin_adamw_tensor& t = tensors[i];
      if (t.numel == 0 || adamw_kind(t) != kind) continue;
      const uint32_t more = (uint32_t)((t.numel + a.chunk - 1) / a.chunk);
      if (a.count == kListed || chunks + more > kMostChunks) launch();
      a.tensor[a.count] = {(uint8_t*)t.param, (const uint8_t*)t.grad, (uint8_t*)t.exp_avg, (uint8_t*)t.exp_avg_sq, t.scales, t.numel};
      a.start[a.count] = chunks;
      a.index[a.count++] = t.index;
      chunks += more;
    }
    launch();
  }
  return optimizer_launched("terra_swin_adamw");
}

}  // namespace
}  // namespace terra

using namespace terra;

extern "C" int terra_swin_gradient_norm_workspace(const terra_swin_tensor* grads, int count) {
  clear_error();
  int64_t partials = 0;
  const int st = grad_counts(grads, count, &partials);
  return st != TERRA_OK ? st : (int)partials;
}

extern "C" int terra_swin_gradient_norm(const terra_swin_tensor* grads, int count, double max_norm, float* result,
                                        double* workspace, void* stream) {
  clear_error();
  int64_t total = 0;
  const int st = grad_counts(grads, count, &total);
  if (st != TERRA_OK) return st;
  if (max_norm != max_norm) return fail(TERRA_ERR_SHAPE, "max_norm is NaN");
  if (result == nullptr || (total > 0 && workspace == nullptr)) return fail(TERRA_ERR_NULL, "result or the workspace is NULL");
  if ((uintptr_t)workspace % 8 != 0 || (uintptr_t)result % 4 != 0) return fail(TERRA_ERR_ALIGN, "result or the workspace is not aligned");
  const uintptr_t w = (uintptr_t)workspace, w_end = w + (uintptr_t)total * 8, r = (uintptr_t)result;
  if (r < w_end && w < r + 12) return fail(TERRA_ERR_SHAPE, "result must not overlap the workspace");
  for (int i = 0; i < count; ++i) {
    const uintptr_t g = (uintptr_t)grads[i].data, elt = dtype_size(grads[i].dtype), end = g + (uintptr_t)grads[i].numel * elt;
    if (grads[i].numel == 0) continue;
    if (g == 0) return fail(TERRA_ERR_NULL, "gradient %d is NULL", i);
    if (g % elt != 0) return fail(TERRA_ERR_ALIGN, "gradient %d is not aligned to its elements", i);
    if ((g < w_end && w < end) || (g < r + 12 && r < end))
      return fail(TERRA_ERR_SHAPE, "result and the workspace must not overlap a gradient");
  }
  hipStream_t s = (hipStream_t)stream;
  GradList a = {};
  a.partials = workspace;
  uint32_t chunks = 0;
  auto launch = [&] {
    if (a.count > 0) gradient_norm_kernel<<<chunks, kNormThreads, 0, s>>>(a);
    a.partials += chunks;
    a.count = 0;
    chunks = 0;
  };
  for (int i = 0; i < count; ++i) {
    if (grads[i].numel == 0) continue;
    const uint32_t more = (uint32_t)((grads[i].numel + kNormChunk - 1) / kNormChunk);
    if (a.count == kGradListed || chunks + more > kMostChunks) launch();
    a.data[a.count] = (const uint8_t*)grads[i].data;
    a.numel[a.count] = grads[i].numel;
    a.dtype[a.count] = (uint8_t)grads[i].dtype;
    a.start[a.count++] = chunks;
    chunks += more;
  }
  launch();
  gradient_norm_result_kernel<<<1, kResultThreads, 0, s>>>(workspace, total, max_norm, result);
  return optimizer_launched("terra_swin_gradient_norm");
}

extern "C" int terra_swin_adamw(const terra_swin_adamw_tensor* tensors, int count, const terra_swin_adamw_desc* desc, void* stream) {
  clear_error();
  try {
    return adamw_checked(tensors, count, desc, (hipStream_t)stream);
  } catch (const std::exception& e) {  // memory for the list of ranges
    return fail(TERRA_ERR_SHAPE, "terra_swin_adamw: %s", e.what());
  }
}
