// What the dropout and residual-norm kernels share: the eight values a lane
// holds of a row, the dropout mask, and sums over lanes and over workgroups.
//
// A chunk is eight columns, the unit of the dropout mask (one Philox call gives
// its eight 16-bit draws).  A lane holds eight values as two halves of four
// columns: one chunk in 16-bit types (16 bytes a load); in fp32 two halves apart,
// neighbouring lanes side by side (16 bytes a load), so that lanes 2i and 2i + 1
// hold the halves of two chunks and share their draws.  kVec: rows of whole,
// 16-byte aligned chunks; otherwise columns are read one by one, or, where
// 16-bit ones stand so, by aligned pairs (GELU backward of 524288 x 766 bf16
// 543 us, x 767 751; a load of 8 or 16 bytes at an address of 2 or 4 took three
// times as long: GELU forward of 2001 x 770 fp16 21 us against 7.5 one by one and
// 5.7 by pairs), halves written at any alignment, and columns from C on are absent.
#pragma once

#include "common.h"

namespace terra {
namespace {

constexpr int kChunkCols = 8;

template <int DT> struct ChunkElt { static constexpr int kBytes = 2; };
template <> struct ChunkElt<TERRA_DTYPE_F32> { static constexpr int kBytes = 4; };

template <int DT>
struct RowChunk {
  static constexpr int kWords = ChunkElt<DT>::kBytes / 2;
  stream_u32x4 q[kWords];
};

// Value j of a chunk in fp32.
template <int DT>
__device__ __forceinline__ float chunk_value(const RowChunk<DT>& r, int j) {
  if constexpr (DT == TERRA_DTYPE_F32) return __uint_as_float(r.q[j >> 2][j & 3]);
  const uint32_t w = r.q[0][j >> 1];
  if constexpr (DT == TERRA_DTYPE_BF16) return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  return __half2float(__ushort_as_half((uint16_t)(j & 1 ? w >> 16 : w & 0xffffu)));
}

typedef __bf16 chunk_bf16x2 __attribute__((ext_vector_type(2)));

// Two fp32 values rounded once, to nearest even, into one word of a 16-bit type.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == TERRA_DTYPE_BF16) {
    chunk_bf16x2 v;
    v[0] = (__bf16)a;
    v[1] = (__bf16)b;
    return __builtin_bit_cast(uint32_t, v);
  } else {
    return (uint32_t)__half_as_ushort(__float2half_rn(a)) | ((uint32_t)__half_as_ushort(__float2half_rn(b)) << 16);
  }
}

// Stores the half at `col` of a row that is not of aligned chunks, rounded once;
// columns from C on are left alone.
template <int DT>
__device__ __forceinline__ void store_half(const float* f, uint8_t* row, int col, int C) {
  if (col >= C) return;
  if constexpr (DT == TERRA_DTYPE_F32) {
    typedef stream_u32x4 __attribute__((aligned(4))) any_u32x4;
    float* p = reinterpret_cast<float*>(row) + col;
    if (col + 4 <= C) {
      *reinterpret_cast<any_u32x4*>(p) =
          stream_u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (col + j < C) p[j] = f[j];
    }
  } else {
    typedef stream_u32x2 __attribute__((aligned(2))) any_u32x2;
    uint16_t* p = reinterpret_cast<uint16_t*>(row) + col;
    if (col + 4 <= C) {
      *reinterpret_cast<any_u32x2*>(p) = stream_u32x2{pack2<DT>(f[0], f[1]), pack2<DT>(f[2], f[3])};
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (col + j < C) p[j] = (uint16_t)pack2<DT>(f[j], 0.f);
    }
  }
}

// ---- the dropout mask --------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011): ten rounds of two 32x32 -> 64-bit products over a
// 128-bit counter under a 64-bit key.  Counter = (column >> 3, row, 0, stream),
// key = the seed; the four result words are the draws of the chunk's eight
// columns, 16 bits each, low half first.  A draw below `threshold` =
// round(p 65536) drops its element, so p is rounded to a multiple of 2^-16, and
// the scale of the kept ones, 65536 / (65536 - threshold), makes the expectation
// exact.  16 bits a draw rather than 32 halve the generator's work, which is as
// long as the memory traffic of a 16-bit element otherwise.
struct DropoutArgs {
  const uint64_t* seed;
  uint32_t threshold;  // 0: nothing is dropped (seed not read); 65536: everything
  float scale;         // of the kept elements (1 without dropout)
  uint32_t stream;
};

struct ChunkDraws {
  uint32_t w[4];
};

__device__ __forceinline__ ChunkDraws chunk_draws(uint64_t seed, uint32_t chunk, uint32_t row, uint32_t stream) {
  uint32_t c0 = chunk, c1 = row, c2 = 0, c3 = stream;
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

__device__ __forceinline__ bool kept(const ChunkDraws& d, int j, uint32_t threshold) {
  return (j & 1 ? d.w[j >> 1] >> 16 : d.w[j >> 1] & 0xffffu) >= threshold;
}

// The value of the neighbouring lane l ^ 1 (quad permute [1, 0, 3, 2]).
__device__ __forceinline__ uint32_t lane_xor1(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false);
}

// The draws of a lane that holds two halves: of chunk `first` in its first
// half and of chunk `second` in the other, the low half of each in an even lane
// and the high half in an odd one.  The even lane draws the first, the odd one
// the second, and they swap.  (An odd lane's columns are beyond an even one's: where
// only the even lane is active, its other half is absent.)
__device__ __forceinline__ ChunkDraws half_draws(uint64_t seed, bool odd, uint32_t first, uint32_t second, uint32_t row,
                                                 uint32_t stream) {
  const ChunkDraws d = chunk_draws(seed, odd ? second : first, row, stream);
  const uint32_t r0 = lane_xor1(odd ? d.w[0] : d.w[2]), r1 = lane_xor1(odd ? d.w[1] : d.w[3]);
  return {{odd ? r0 : d.w[0], odd ? r1 : d.w[1], odd ? d.w[2] : r0, odd ? d.w[3] : r1}};
}

// ---- sums over the lanes of a row ---------------------------------------------
// Sum over the kL aligned lanes of a wave (kL = 8, 16, 32 or 64); every lane ends
// with the same bits, since each step adds the same two values on both sides.
template <int kL>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (kL == 8) return group8_sum(v);
  v = row16_sum(v);
  if constexpr (kL >= 32) {
    const uint32_t b = __float_as_uint(v);
    const auto p = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (kL >= 64) {
    const uint32_t b = __float_as_uint(v);
    const auto p = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

// Sums over the kG lanes of a row: of a part of a wave (kG <= 64), or of the
// whole workgroup (kG = its threads), whose waves meet in LDS.  Two slots take
// turns, so one barrier a sum is enough: a wave writes a slot again only after
// the barrier of the sum in between, which every wave reaches after it has
// read that slot.
template <int kG>
struct RowSum {
  static constexpr int kWaves = kG > 64 ? kG / 64 : 1;
  struct Shared { float part[kG > 64 ? 2 : 1][kWaves][2]; };
  Shared* s;
  int turn = 0;

  __device__ __forceinline__ explicit RowSum(Shared* shared) : s(shared) {}

  __device__ __forceinline__ void two(float& a, float& b) {
    if constexpr (kG <= 64) {
      a = lanes_sum<kG>(a);
      b = lanes_sum<kG>(b);
    } else {
      a = lanes_sum<64>(a);
      b = lanes_sum<64>(b);
      if ((threadIdx.x & 63) == 0) {
        s->part[turn][threadIdx.x >> 6][0] = a;
        s->part[turn][threadIdx.x >> 6][1] = b;
      }
      lds_sync();
      const float* p = s->part[turn][threadIdx.x % kWaves];  // one wave's sums a lane, then over those lanes
      a = waves_sum(p[0]);
      b = waves_sum(p[1]);
      turn ^= 1;
    }
  }
  __device__ __forceinline__ float one(float a) {
    if constexpr (kG <= 64) return lanes_sum<kG>(a);
    float b = 0.f;
    two(a, b);
    return a;
  }
  static __device__ __forceinline__ float waves_sum(float v) {
    static_assert(kG <= 64 || kWaves == 4 || kWaves == 8, "waves of a row");
    if constexpr (kWaves == 8) return group8_sum(v);
    v += dpp_move<0xb1>(v);
    return v + dpp_move<0x4e>(v);
  }
  // A workgroup barrier that waits for LDS only: loads of rows ahead stay in flight.
  static __device__ __forceinline__ void lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
};

// ---- column sums in two levels -------------------------------------------------
// Adds up partial sums of the workgroups of an earlier launch, in an order
// that the sizes alone fix: dst[b][c] = sum over i < count of
// src[(b * count + i) * src_stride + c].
struct SumJob {
  const float* src;
  float* dst;
  int64_t src_stride;
  int32_t count;
  int32_t batch;
};
constexpr int kMaxSumJobs = 5;
struct SumJobs {
  SumJob job[kMaxSumJobs];
  int32_t C;
};

constexpr int kSumThreads = 1024;
constexpr int kSumCols = 16;
constexpr int kSumParts = kSumThreads / kSumCols;

constexpr int kSumGrid = 1 << 21;  // workgroups a dimension: a grid holds fewer than 2^32 threads in each

// One workgroup for 16 columns of one row of one job: 64 adders take every
// 64th partial each, in fp64.  (static: each source file that sums has its own
// copy.)  Few columns a workgroup, so that a vector of some hundred columns
// still has tens of workgroups to wait for the partials' loads.
static __global__ __launch_bounds__(kSumThreads) void sum_partials_kernel(const SumJobs jobs) {
  const SumJob j = jobs.job[blockIdx.y];
  __shared__ double s[kSumParts][kSumCols];
  const int lane = threadIdx.x % kSumCols, part = threadIdx.x / kSumCols;
  for (int first = blockIdx.x * kSumCols; first < jobs.C; first += gridDim.x * kSumCols) {
    const int c = first + lane;
    for (int b = blockIdx.z; b < j.batch; b += gridDim.z) {
      double sum = 0.0;
      const float* src = j.src + (int64_t)b * j.count * j.src_stride + (c < jobs.C ? c : 0);
      constexpr int kAhead = 8;
      for (int i = part; i < j.count; i += kAhead * kSumParts) {
        float v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
          const int at = i + u * kSumParts;
          v[u] = src[(int64_t)(at < j.count ? at : i) * j.src_stride];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) sum += i + u * kSumParts < j.count ? (double)v[u] : 0.0;
      }
      s[part][lane] = sum;
      __syncthreads();
      for (int half = kSumParts / 2; half > 0; half /= 2) {
        if (part < half) s[part][lane] = sum += s[part + half][lane];
        __syncthreads();
      }
      if (part == 0 && c < jobs.C) j.dst[(int64_t)b * jobs.C + c] = (float)sum;
    }
  }
}

// Launches the jobs with a destination (count of them in `n`).
inline void launch_sums(const SumJobs& jobs, int n, hipStream_t s) {
  int batch = 1;
  for (int i = 0; i < n; ++i) batch = jobs.job[i].batch > batch ? jobs.job[i].batch : batch;
  const int groups = (jobs.C + kSumCols - 1) / kSumCols;  // of columns
  const dim3 grid((unsigned)(groups < kSumGrid ? groups : kSumGrid), (unsigned)n, (unsigned)(batch < 1024 ? batch : 1024));
  sum_partials_kernel<<<grid, kSumThreads, 0, s>>>(jobs);
}

// Whether dropout with these arguments is valid; fills `d`.
inline int dropout_args(double p, const void* seed, uint32_t stream, DropoutArgs* d) {
  if (!(p >= 0.0 && p <= 1.0)) return fail(TERRA_ERR_SHAPE, "the dropout probability must be in [0, 1] (got %g)", p);
  d->threshold = (uint32_t)(p * 65536.0 + 0.5);
  d->scale = d->threshold < 65536u ? (float)(65536.0 / (65536.0 - (double)d->threshold)) : 0.f;
  d->stream = stream;
  d->seed = (const uint64_t*)seed;
  if (d->threshold > 0 && seed == nullptr) return fail(TERRA_ERR_NULL, "dropout needs a seed");
  if (((uintptr_t)seed & 7u) != 0) return fail(TERRA_ERR_ALIGN, "the seed must be 8-byte aligned");
  return TERRA_OK;
}

}  // namespace
}  // namespace terra
