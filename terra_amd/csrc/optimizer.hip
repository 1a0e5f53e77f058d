// The update of the parameters: the norm of all gradients as one vector, and
// an AdamW step over many tensors at once, its moments in 32 bits or in 8
// (the formulas stand at the entry points' declarations).
//
// The tensors of a launch are listed in its arguments, up to kListed of them,
// so nothing has to be copied to the device before it and a captured graph
// keeps them; a workgroup has a chunk of one tensor, found by a binary search.
#include "row_chunk.h"

#include <algorithm>
#include <exception>
#include <initializer_list>
#include <vector>

namespace terra {
namespace {

constexpr int kListed = 64;  // tensors of a launch: 48 bytes each, of 4 KB of arguments

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

struct GradList {
  const uint8_t* data[kListed];
  int64_t numel[kListed];
  uint32_t start[kListed];
  int32_t dtype[kListed];
  double* partials;
  int32_t count;
};

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
  return v;
}

// The thread's sum of squares of elements begin .. end - 1.
template <int DT>
__device__ __forceinline__ double squares(const uint8_t* g, int64_t begin, int64_t end) {
  double sum = 0.0;
  const bool vec = (uintptr_t)g % (4 * ChunkElt<DT>::kBytes) == 0;
  int64_t i = begin + threadIdx.x * 4;
  if (vec)
    for (; i + 4 <= end; i += kNormThreads * 4) {
      float f[4];
      four_values<DT, true>(g, i, 4, f);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fma((double)f[j], (double)f[j], sum);
    }
  for (; i < end; i += kNormThreads * 4) {
    float f[4];
    four_values<DT, false>(g, i, (int)(end - i < 4 ? end - i : 4), f);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fma((double)f[j], (double)f[j], sum);
  }
  return sum;
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
constexpr int64_t kAdamChunk = 8192;  // elements of a workgroup
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
  float keep, rate, root, eps;  // 1 - lr decay, lr / (1 - beta1^t), 1 / (1 - beta2^t), eps
  float factor;                 // of the gradients
  uint32_t step;

  __device__ __forceinline__ explicit AdamStep(const AdamList& a) {
    const int64_t t = a.step_ptr != nullptr ? *a.step_ptr : a.step;
    const double lr = a.lr_ptr != nullptr ? (double)*a.lr_ptr : a.lr;
    keep = (float)(1.0 - lr * a.decay);
    rate = (float)(lr / (1.0 - power(a.beta1, t)));
    root = (float)(1.0 / (1.0 - power(a.beta2, t)));
    eps = (float)a.eps;
    factor = a.grad_factor != nullptr ? *a.grad_factor : 1.f;
    if (a.maximize) factor = -factor;
    step = (uint32_t)t;
  }
  __device__ __forceinline__ float updated(float p, float m, float v) const {
    return p * keep - rate * (m / (sqrtf(v * root) + eps));
  }
};

template <int DTP, int DTG, bool kVec>
__device__ __forceinline__ void adam_elements(const AdamEntry& e, const AdamStep& st, float b1, float c1, float b2, float c2,
                                              int64_t i, int n) {
  float p[4], g[4], m[4], v[4];
  four_values<DTP, kVec>(e.param, i, n, p);
  four_values<DTG, kVec>(e.grad, i, n, g);
  four_values<TERRA_DTYPE_F32, kVec>(e.first, i, n, m);
  four_values<TERRA_DTYPE_F32, kVec>(e.second, i, n, v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float d = g[j] * st.factor;
    m[j] = fmaf(c1, d, b1 * m[j]);
    v[j] = fmaf(c2 * d, d, b2 * v[j]);
    p[j] = st.updated(p[j], m[j], v[j]);
  }
  put_four<DTP, kVec>(e.param, i, n, p);
  put_four<TERRA_DTYPE_F32, kVec>(e.first, i, n, m);
  put_four<TERRA_DTYPE_F32, kVec>(e.second, i, n, v);
}

template <int DTP, int DTG>
__global__ __launch_bounds__(kAdamThreads) void adamw_kernel(const AdamList a) {
  if (a.found_inf != nullptr && *a.found_inf != 0.f) return;
  const int t = tensor_of(a.start, a.count, blockIdx.x);
  const AdamEntry e = a.tensor[t];
  const AdamStep st(a);
  const float b1 = (float)a.beta1, c1 = (float)(1.0 - a.beta1), b2 = (float)a.beta2, c2 = (float)(1.0 - a.beta2);
  const int64_t begin = (int64_t)(blockIdx.x - a.start[t]) * kAdamChunk;
  const int64_t end = begin + kAdamChunk < e.numel ? begin + kAdamChunk : e.numel;
  const bool vec = (uintptr_t)e.param % (4 * ChunkElt<DTP>::kBytes) == 0 && (uintptr_t)e.grad % (4 * ChunkElt<DTG>::kBytes) == 0 &&
                   ((uintptr_t)e.first | (uintptr_t)e.second) % 16 == 0;
  int64_t i = begin + threadIdx.x * 4;
  if (vec)
    for (; i + 4 <= end; i += kAdamThreads * 4) adam_elements<DTP, DTG, true>(e, st, b1, c1, b2, c2, i, 4);
  for (; i < end; i += kAdamThreads * 4)
    adam_elements<DTP, DTG, false>(e, st, b1, c1, b2, c2, i, (int)(end - i < 4 ? end - i : 4));
}

// ---- moments in 8 bits ----------------------------------------------------------
// In 64 bits up to the codes: a value next to the border of two codes goes to
// the one that the formula says.

__device__ __forceinline__ uint32_t fp8_code(float v) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.f, 0, false) & 0xffu; }
__device__ __forceinline__ float fp8_value(uint32_t code) { return __builtin_amdgcn_cvt_f32_fp8((int)code, 0); }

// y (at most 448 and a little in size) to the nearest code of e4m3. Rounded to 32
// bits towards odd first, so that the second rounding sees on which side of a border it is.
__device__ __forceinline__ uint32_t nearest_code(double y) {
  if (y != y) return 0x7fu;
  float f = (float)y;
  const double back = (double)f;
  uint32_t b = __float_as_uint(f);
  if (back != y && (b & 1u) == 0) b += (fabs(back) > fabs(y)) ? ~0u : 1u;  // to the odd neighbour on y's side
  f = __uint_as_float(b);
  f = fminf(fmaxf(f, -448.f), 448.f);
  return fp8_code(f);
}

// w = v / scale^2: one of the codes next to its root, see terra_swin_adamw.
__device__ __forceinline__ uint32_t root_code(double w, uint32_t draw) {
  if (!(w > 0.0)) return 0u;
  const float r = fminf(sqrtf((float)w), 448.f);
  const int exponent = max((int)(__float_as_uint(r) >> 23) - 127, -6);
  const float grid = __uint_as_float((uint32_t)(exponent - 3 + 127) << 23);
  const float low = floorf(r / grid) * grid, high = low + grid;
  const double span = (double)high * high - (double)low * low;
  const bool up = w - (double)low * low > ((double)draw + 0.5) * (1.0 / 65536.0) * span && low < 448.f;
  return fp8_code(fmaxf(up ? high : low, 0.001953125f));
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

// A wave takes blocks of 256 elements, four a lane.
template <int DTP, int DTG>
__global__ __launch_bounds__(kAdamThreads) void adamw_8bit_kernel(const AdamList a) {
  if (a.found_inf != nullptr && *a.found_inf != 0.f) return;
  const int t = tensor_of(a.start, a.count, blockIdx.x);
  const AdamEntry e = a.tensor[t];
  const AdamStep st(a);
  const uint64_t seed = *a.seed;
  const double factor = (double)st.factor, b1 = a.beta1, c1 = 1.0 - a.beta1, b2 = a.beta2, c2 = 1.0 - a.beta2;
  const int64_t blocks = (e.numel + kScaled - 1) / kScaled;
  const int64_t begin = (int64_t)(blockIdx.x - a.start[t]) * (kAdamChunk / kScaled);
  const int64_t end = begin + kAdamChunk / kScaled < blocks ? begin + kAdamChunk / kScaled : blocks;
  const int lane = threadIdx.x & 63;
  const bool vec = (uintptr_t)e.param % (4 * ChunkElt<DTP>::kBytes) == 0 && (uintptr_t)e.grad % (4 * ChunkElt<DTG>::kBytes) == 0 &&
                   ((uintptr_t)e.first | (uintptr_t)e.second) % 4 == 0;
  for (int64_t b = begin + (threadIdx.x >> 6); b < end; b += kAdamThreads / 64) {
    const int64_t i = b * kScaled + lane * 4, left = e.numel - i;
    const int n = left >= 4 ? 4 : left > 0 ? (int)left : 0;
    const bool whole = vec && n == 4;
    float p[4], g[4];
    uint32_t mc = 0, rc = 0;
    if (whole) {
      four_values<DTP, true>(e.param, i, 4, p);
      four_values<DTG, true>(e.grad, i, 4, g);
      mc = *reinterpret_cast<const uint32_t*>(e.first + i);
      rc = *reinterpret_cast<const uint32_t*>(e.second + i);
    } else {
      four_values<DTP, false>(e.param, i, n, p);
      four_values<DTG, false>(e.grad, i, n, g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mc |= j < n ? (uint32_t)e.first[i + j] << (8 * j) : 0u;
        rc |= j < n ? (uint32_t)e.second[i + j] << (8 * j) : 0u;
      }
    }
    const double sm = (double)e.scales[b], sr = (double)e.scales[blocks + b];
    double m[4], v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double d = (double)g[j] * factor;
      const double r = (double)fp8_value((rc >> (8 * j)) & 0xffu) * sr;
      m[j] = b1 * ((double)fp8_value((mc >> (8 * j)) & 0xffu) * sm) + c1 * d;
      v[j] = b2 * (r * r) + c2 * (d * d);
      p[j] = st.updated(p[j], (float)m[j], (float)v[j]);
    }
    // The scales: 32-bit roundings of the largest values, which are taken in 64.  With an infinity or a NaN
    // the scale is infinite, and all of the block NaN when it is read again.
    double big_m = 0.0, big_v = 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      big_m = fmax(big_m, fabs(m[j]));
      big_v = fmax(big_v, v[j]);
      if (!(fabs(m[j]) <= 1.7976931348623157e308)) big_m = __builtin_inf();
      if (!(v[j] <= 1.7976931348623157e308)) big_v = __builtin_inf();
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
      big_m = fmax(big_m, __shfl_xor(big_m, d));
      big_v = fmax(big_v, __shfl_xor(big_v, d));
    }
    const float new_m = (float)(big_m / 448.0), new_r = (float)(sqrt(big_v) / 448.0);
    const double inv_m = new_m > 0.f ? 1.0 / (double)new_m : 0.0, inv_r = new_r > 0.f ? 1.0 / (double)new_r : 0.0;
    const uint32_t chunk = (uint32_t)(i >> 3);
    const ChunkDraws dr = adam_draws(seed, chunk, a.index[t], st.step, a.stream);
    uint32_t out_m = 0, out_r = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = lane & 1 ? dr.w[2 + (j >> 1)] : dr.w[j >> 1];
      out_m |= nearest_code(m[j] * inv_m) << (8 * j);
      out_r |= root_code(v[j] * inv_r * inv_r, j & 1 ? w >> 16 : w & 0xffffu) << (8 * j);
    }
    if (whole) {
      put_four<DTP, true>(e.param, i, 4, p);
      *reinterpret_cast<uint32_t*>(e.first + i) = out_m;
      *reinterpret_cast<uint32_t*>(e.second + i) = out_r;
    } else {
      put_four<DTP, false>(e.param, i, n, p);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) {
          e.first[i + j] = (uint8_t)(out_m >> (8 * j));
          e.second[i + j] = (uint8_t)(out_r >> (8 * j));
        }
    }
    if (lane == 0) {
      e.scales[b] = new_m;
      e.scales[blocks + b] = new_r;
    }
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
      const uint32_t more = (uint32_t)((t.numel + kAdamChunk - 1) / kAdamChunk);
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
    if (a.count == kListed || chunks + more > kMostChunks) launch();
    a.data[a.count] = (const uint8_t*)grads[i].data;
    a.numel[a.count] = grads[i].numel;
    a.dtype[a.count] = grads[i].dtype;
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
