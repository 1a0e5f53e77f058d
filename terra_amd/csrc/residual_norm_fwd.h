// Forward of the end of a half-block (residual_norm.h): the branch's
// post-norm, dropout, gate, scaled residual and the next half-block's norm in
// one pass.  Bound by memory: h and x read once, y and z written once.
#pragma once

#include "residual_norm.h"

namespace terra {
namespace {

template <int DTH, int DTX, int kG, int kK, bool kVec, int kF>
__global__ __launch_bounds__(tail_threads(kG)) void tail_kernel(const TailArgs a) {
  constexpr int kGroups = tail_threads(kG) / kG;
  constexpr int kHB = ChunkElt<DTH>::kBytes, kXB = ChunkElt<DTX>::kBytes;
  constexpr int kP = DTX == TERRA_DTYPE_F32 ? 4 : 8;
  using Params = ColumnParams<4, kG, kK, kP>;
  __shared__ typename RowSum<kG>::Shared s_red;
  __shared__ typename Params::Shared s_par;
  const int group = threadIdx.x / kG, C = a.C;
  const RowLanes<kG, kK, kP> at = {(int)(threadIdx.x % kG), C};
  RowSum<kG> sum(&s_red);
  const bool full = C == kG * kK * kChunkCols;  // every lane has columns
  constexpr bool kPairs = kF & kTailPairs;
  Params par(&s_par);  // gw, gb (branch_params), nw, nb
  const uint64_t seed = tail_has<kF>(a, kTailDrop) ? *a.drop.seed : 0;
  // A row's chunks of h and x; a row past the end re-reads the last one.
  struct Row {
    uint32_t r;
    bool has;
    RowChunk<DTH> h[kK];
    RowChunk<DTX> x[kK];
  };
  auto fetch = [&](uint32_t base) {
    Row q;
    const uint32_t row = base + group;
    q.r = row < a.rows ? row : a.rows - 1;
    const int64_t src = a.flags & kTailWindows ? a.map.source(q.r) : (int64_t)q.r;
    q.has = src >= 0;
    const uint8_t* hp = a.h + (q.has ? src : 0) * a.h_row_bytes;
    const uint8_t* xp = a.x + (int64_t)q.r * a.x_row_bytes;
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      q.h[k] = at.template load<DTH, kVec, kPairs>(hp, k);
      q.x[k] = at.template load<DTX, kVec, kPairs>(xp, k);
    }
    return q;
  };
  const uint32_t step = gridDim.x * kGroups;
  uint32_t base = blockIdx.x * kGroups;
  Row ahead = fetch(base);
  par.fill(at, [&](int c, float (&v)[4]) {
    branch_params(a, a.gate_rows == 1 ? a.gate : nullptr, c, v[0], v[1]);
    v[2] = param_at(a.nw, 1.f, c);
    v[3] = param_at(a.nb, 0.f, c);
  });
  if constexpr (Params::kLds) RowSum<kG>::lds_sync();
  for (; base < a.rows; base += step) {
    par.stay();
    const Row q = ahead;
    if (base + step < a.rows) ahead = fetch(base + step);
    const uint32_t r = q.r;
    const bool live = base + group < a.rows, has = q.has;
    float v[kK][kChunkCols];
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      at.template values<DTH, kVec>(q.h[k], k, has, full && !(a.flags & kTailWindows), v[k]);
    }
    if (tail_has<kF>(a, kTailPost)) normalise<kG, kK, kP, kVec>(v, a.flags & kTailPostLayer, a.post_eps, a.inv_c, at, sum);
    const uint32_t live_rows = min(a.rows - base, (uint32_t)kGroups);
    const __amdgpu_buffer_rsrc_t y_out = buffer_rsrc(a.y + (int64_t)base * C * kXB, live_rows * (uint32_t)(C * kXB));
#pragma unroll
    for (int k = 0; k < kK; ++k) {
      float gw[kChunkCols], gb[kChunkCols], xv[kChunkCols];
      par.get(0, k, at, gw);
      par.get(1, k, at, gb);
      if (a.gate_rows > 1) {  // this row's sample's gate
        const float* gate = a.gate + (int64_t)(r / a.per_sample) * C;
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const float g = at.template has<kVec>(k, j) ? gate[at.base(k, j >> 2) + (j & 3)] : 0.f;
          gw[j] *= g;
          gb[j] *= g;
        }
      }
      at.template values<DTX, kVec>(q.x[k], k, true, full, xv);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) v[k][j] = has ? fmaf(v[k][j], gw[j], gb[j]) : 0.f;
      const ChunkDraws d = at.draws(tail_has<kF>(a, kTailDrop), seed, k, r, a.drop.stream);
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j)
        v[k][j] = fmaf(a.alpha, xv[j], kept(d, j, a.drop.threshold) ? v[k][j] : 0.f);
      if (live) at.template store<DTX, kVec>(v[k], y_out, (uint32_t)(group * C) * kXB, a.y + (int64_t)r * C * kXB, k);
    }
    if (tail_has<kF>(a, kTailNext)) {
      normalise<kG, kK, kP, kVec>(v, a.flags & kTailNextLayer, a.next_eps, a.inv_c, at, sum);
      const __amdgpu_buffer_rsrc_t z_out = buffer_rsrc(a.z + (int64_t)base * C * kHB, live_rows * (uint32_t)(C * kHB));
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        float w[kChunkCols], b[kChunkCols];
        par.get(2, k, at, w);
        par.get(3, k, at, b);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) v[k][j] = fmaf(v[k][j], w[j], b[j]);
        if (live) at.template store<DTH, kVec>(v[k], z_out, (uint32_t)(group * C) * kHB, a.z + (int64_t)r * C * kHB, k);
      }
    }
  }
}

template <int DTH, int DTX, int kG, int kK, bool kVec, int kF>
void launch_fwd(const TailArgs& a, hipStream_t s) {
  constexpr uint32_t kGroups = tail_threads(kG) / kG;
  // Row groups of a workgroup: few, so that workgroups that load and such that
  // compute are always side by side (2048 that stay for all rows: 148 us at
  // 524288 x 192 bf16, one group each 131), but enough for the parameters, 16 C
  // bytes a workgroup, to be a small part of what it reads.
  constexpr uint32_t kTurns = kG > 64 ? 16 : (kG > 16 ? kG / 16 : 1);
  const uint32_t need = (a.rows + kGroups - 1) / kGroups, blocks = (need + kTurns - 1) / kTurns;
  constexpr uint32_t kMost = 1u << 22;  // a grid holds fewer than 2^32 threads
  tail_kernel<DTH, DTX, kG, kK, kVec, kF><<<blocks < kMost ? blocks : kMost, tail_threads(kG), 0, s>>>(a);
}

template <int DTH, int DTX>
void dispatch_fwd(const TailArgs& a, bool vec, hipStream_t s) {
  TERRA_TAIL_SHAPES(launch_fwd, tail_shape(a.C, tail_pieces(DTX), 3), 3, a.flags, vec, a, s)
}

}  // namespace
}  // namespace terra
