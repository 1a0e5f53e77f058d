// Backward of the end of a half-block (residual_norm.h), from the gradients
// of y and z.  No statistic, mask or intermediate of the forward is kept: each
// row is recomputed from h and x in registers, and then, with gw = gate s w1
// and gb = gate s b1 (branch_params),
//
//   y  = alpha x + keep (nhat gw + gb)
//   g  = dz w2,  dY = dy + r2 (g - mean g - yhat mean(g yhat)),  dx = alpha dY
//   t  = keep dY,  u = t gw,  dh = r1 (u - mean u - nhat mean(u nhat))
//   dw2 = sum dz yhat,  db2 = sum dz
//
// (an RMS norm has no mean g and mean u term; without a norm dY = dy, dh = u).
// The branch's three parameter gradients are two sums over the rows that share
// a gate, A = s sum t nhat and B = s sum t:
//   dgate = w1 A + b1 B,  dw1 = sum over gates of gate A,  db1 = ... gate B
// which spares the rows' loop a sum, the value m and a product per element.
// Bound by memory: h, x, dy, dz read once, dh and dx written once.
//
// Sums over rows: a unit is every slabs-th group of rows of one sample (so
// that workgroups side by side read rows side by side; with a run of rows each,
// 156672 x 1024 bf16 took 402 us, 363 so), workgroups take units in grid strides, and
// each lane keeps the sums of its columns in registers; A and B leave them unit by unit, since the gate changes
// with the sample.  A second launch adds the workgroups' sums
// (sum_partials_kernel): no atomics, an order that the sizes fix.
#pragma once

#include "residual_norm.h"

namespace terra {
namespace {

// Waves a SIMD that the registers of a kernel must leave room for: two where it
// would otherwise take a few more than half of them (131072 x 768, bf16 h and
// fp32 x: 353 us, with one wave 421); columns read one by one are slower so
// (262144 x 385 bf16: 599 us against 505).
template <int DTX, int kG, int kK, bool kVec, int kF>
constexpr int tail_bwd_waves() {
  if (kG == 512 && kK == 1) return 4;
  return kK == 3 || (kF & kTailPairs) != 0 || (kVec && kG == 64 && DTX == TERRA_DTYPE_F32) ? 2 : 1;
}

template <int DTH, int DTX, int kG, int kK, bool kVec, int kF>
__global__ __launch_bounds__(tail_threads(kG), (tail_bwd_waves<DTX, kG, kK, kVec, kF>())) void tail_bwd_kernel(const TailArgs a) {
  constexpr int kThreads = tail_threads(kG), kGroups = kThreads / kG, kCols = kG * kK * kChunkCols;
  constexpr int kHB = ChunkElt<DTH>::kBytes, kXB = ChunkElt<DTX>::kBytes;
  constexpr int kP = DTX == TERRA_DTYPE_F32 ? 4 : 8;
  using Params = ColumnParams<3, kG, kK, kP>;
  __shared__ typename RowSum<kG>::Shared s_red;
  __shared__ typename Params::Shared s_par;
  __shared__ __attribute__((aligned(16))) float s_acc[kGroups > 1 ? kGroups * kCols : 1];
  const int group = threadIdx.x / kG, C = a.C;
  const RowLanes<kG, kK, kP> at = {(int)(threadIdx.x % kG), C};
  RowSum<kG> sum(&s_red);
  const bool full = C == kG * kK * kChunkCols;  // every lane has columns
  constexpr bool kPairs = kF & kTailPairs;
  Params par(&s_par);  // gw, gb, w2
  // Returns whether a gate is infinite or NaN: only then do the rows' loops see
  // to it that a dropped element's gradient is 0 (with the test in every case,
  // 262144 x 384 bf16 took 274 us instead of 243).
  auto stage = [&](const float* gate) {
    int odd = 0;
    par.fill(at, [&](int c, float (&v)[3]) {
      branch_params(a, gate, c, v[0], v[1]);
      v[2] = param_at(a.nw, 1.f, c);
      odd |= !(fabsf(v[0]) <= 3.4028235e38f);
    });
    if (!tail_has<kF>(a, kTailDrop)) odd = 0;
    return __syncthreads_or(odd) != 0;
  };
  bool odd_gate = stage(a.gate_rows == 1 ? a.gate : nullptr);
  const uint64_t seed = tail_has<kF>(a, kTailDrop) ? *a.drop.seed : 0;

  float acc_a[kK][kChunkCols] = {}, acc_b[kK][kChunkCols] = {}, acc_nw[kK][kChunkCols] = {}, acc_nb[kK][kChunkCols] = {};
  // The workgroup's sums of two vectors over its row groups, given to f(column, sum, other).
  constexpr int kOwn = (kCols + kThreads - 1) / kThreads;
  auto flush = [&](float (&p)[kK][kChunkCols], float (&q)[kK][kChunkCols], auto f) {
    if constexpr (kGroups > 1) {
      float own[2][kOwn];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          const float* v = which == 0 ? p[k] : q[k];
          *reinterpret_cast<float4*>(&s_acc[group * kCols + at.base(k, 0)]) = make_float4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<float4*>(&s_acc[group * kCols + at.base(k, 1)]) = make_float4(v[4], v[5], v[6], v[7]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int c = threadIdx.x + i * kThreads;
          float t = 0.f;
          if (c < kCols)
#pragma unroll
            for (int g = 0; g < kGroups; ++g) t += s_acc[g * kCols + c];
          own[which][i] = t;
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int c = threadIdx.x + i * kThreads;
        if (c < C) f(c, own[0][i], own[1][i]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const int c = at.base(k, j >> 2) + (j & 3);
          if (c < C) f(c, p[k][j], q[k][j]);
        }
    }
  };
  float* const mine = a.partial != nullptr ? a.partial + (int64_t)blockIdx.x * 4 * C : nullptr;

  for (uint32_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
    const uint32_t sample = unit / a.slabs, slab = unit % a.slabs;
    const uint32_t end = (sample + 1) * a.per_sample;
    const float* const gate = a.gate_rows > 0 ? a.gate + (int64_t)sample * C : nullptr;
    if (a.gate_rows > 1) {
      if constexpr (Params::kLds) __syncthreads();
      odd_gate = stage(gate);
    }
    for (uint32_t base = sample * a.per_sample + slab * kGroups; base < end; base += a.slabs * kGroups) {
      par.stay();
      const uint32_t row = base + group;
      const bool live = row < end;
      const uint32_t r = live ? row : end - 1;  // a row past the end re-reads the sample's last one
      const int64_t src = a.flags & kTailWindows ? a.map.source(r) : (int64_t)r;
      const bool has = src >= 0;
      RowChunk<DTH> hq[kK], dzq[kK];
      RowChunk<DTX> xq[kK], dyq[kK];
      const uint8_t* hp = a.h + (has ? src : 0) * a.h_row_bytes;
      const uint8_t* xp = a.x + (int64_t)r * a.x_row_bytes;
      const uint8_t* dyp = a.flags & kTailDy ? a.dy + (int64_t)r * C * kXB : xp;
      const uint8_t* dzp = tail_has<kF>(a, kTailNext) ? a.dz + (int64_t)r * C * kHB : hp;
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        hq[k] = at.template load<DTH, kVec, kPairs>(hp, k);
        xq[k] = at.template load<DTX, kVec, kPairs>(xp, k);
        dzq[k] = at.template load<DTH, kVec, kPairs>(dzp, k);
        dyq[k] = at.template load<DTX, kVec, kPairs>(dyp, k);
      }
      // The forward: nhat in nv, y in yv.
      float nv[kK][kChunkCols], yv[kK][kChunkCols], dv[kK][kChunkCols];
      ChunkDraws draws[kK];
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        at.template values<DTH, kVec>(hq[k], k, has, full && !(a.flags & kTailWindows), nv[k]);
      }
      float r1 = 1.f;
      if (tail_has<kF>(a, kTailPost)) r1 = normalise<kG, kK, kP, kVec>(nv, a.flags & kTailPostLayer, a.post_eps, a.inv_c, at, sum);
#pragma unroll
      for (int k = 0; k < kK; ++k) draws[k] = at.draws(tail_has<kF>(a, kTailDrop), seed, k, r, a.drop.stream);
      if (!tail_has<kF>(a, kTailPost) && tail_has<kF>(a, kTailDrop))  // NaN and infinities of the branch stay out of A where they are dropped
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) nv[k][j] = kept(draws[k], j, a.drop.threshold) ? nv[k][j] : 0.f;
      if (tail_has<kF>(a, kTailNext)) {
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          float gw[kChunkCols], gb[kChunkCols], xv[kChunkCols];
          par.get(0, k, at, gw);
          par.get(1, k, at, gb);
          at.template values<DTX, kVec>(xq[k], k, true, full, xv);
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j)
            yv[k][j] = fmaf(a.alpha, xv[j], has && kept(draws[k], j, a.drop.threshold) ? fmaf(nv[k][j], gw[j], gb[j]) : 0.f);
        }
        const float r2 = normalise<kG, kK, kP, kVec>(yv, a.flags & kTailNextLayer, a.next_eps, a.inv_c, at, sum);
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          float w[kChunkCols];
          par.get(2, k, at, w);
          at.template values<DTH, kVec>(dzq[k], k, true, full, dv[k]);
          if (live)
#pragma unroll
            for (int j = 0; j < kChunkCols; ++j) {
              acc_nw[k][j] = fmaf(dv[k][j], yv[k][j], acc_nw[k][j]);
              acc_nb[k][j] += dv[k][j];
            }
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) {
            dv[k][j] *= w[j];
            s0 += dv[k][j];
            s1 = fmaf(dv[k][j], yv[k][j], s1);
          }
        }
        sum.two(s0, s1);
        s0 = a.flags & kTailNextLayer ? r2 * (s0 * a.inv_c) : 0.f;
        s1 = r2 * (s1 * a.inv_c);
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          float dyv[kChunkCols];
          at.template values<DTX, kVec>(dyq[k], k, true, full, dyv);
          if (!(a.flags & kTailDy))
#pragma unroll
            for (int j = 0; j < kChunkCols; ++j) dyv[j] = 0.f;
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) dv[k][j] = fmaf(r2, dv[k][j], fmaf(-s1, yv[k][j], dyv[j] - s0));
        }
      } else {
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          at.template values<DTX, kVec>(dyq[k], k, true, full, dv[k]);
          if (!(a.flags & kTailDy))
#pragma unroll
            for (int j = 0; j < kChunkCols; ++j) dv[k][j] = 0.f;
        }
      }
      // dv is dY: dx, then t, A and B, then u in dv.
      const __amdgpu_buffer_rsrc_t dx_out =
          buffer_rsrc(a.dx + (int64_t)base * C * kXB, min(end - base, (uint32_t)kGroups) * (uint32_t)(C * kXB));
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        float out[kChunkCols], gw[kChunkCols];
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) out[j] = a.alpha * dv[k][j];
        if (live) at.template store<DTX, kVec>(out, dx_out, (uint32_t)(group * C) * kXB, a.dx + (int64_t)r * C * kXB, k);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) dv[k][j] = kept(draws[k], j, a.drop.threshold) ? dv[k][j] : 0.f;
        if (live && has)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) {
            acc_a[k][j] = fmaf(dv[k][j], nv[k][j], acc_a[k][j]);
            acc_b[k][j] += dv[k][j];
          }
        par.get(0, k, at, gw);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) dv[k][j] *= gw[j];
        if (odd_gate)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) dv[k][j] = kept(draws[k], j, a.drop.threshold) ? dv[k][j] : 0.f;
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          s0 += dv[k][j];
          s1 = fmaf(dv[k][j], nv[k][j], s1);
        }
      }
      if (tail_has<kF>(a, kTailPost)) {
        sum.two(s0, s1);
        s0 = a.flags & kTailPostLayer ? r1 * (s0 * a.inv_c) : 0.f;
        s1 = r1 * (s1 * a.inv_c);
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) dv[k][j] = fmaf(r1, dv[k][j], fmaf(-s1, nv[k][j], -s0));
      }
      // In window order each row has a place of its own: a descriptor for it
      // would not be uniform over the wave's rows.
      if (a.flags & kTailWindows) {
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          if (live && has) at.template store<DTH, kVec>(dv[k], a.dh + src * C * kHB, k);
        }
      } else {
        const __amdgpu_buffer_rsrc_t dh_out =
            buffer_rsrc(a.dh + (int64_t)base * C * kHB, min(end - base, (uint32_t)kGroups) * (uint32_t)(C * kHB));
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          if (live) at.template store<DTH, kVec>(dv[k], dh_out, (uint32_t)(group * C) * kHB, a.dh + (int64_t)r * C * kHB, k);
        }
      }
    }
    if (a.branch_sums) {
      const bool first = unit == blockIdx.x;
      flush(acc_a, acc_b, [&](int c, float sa, float sb) {
        sa *= a.drop.scale;
        sb *= a.drop.scale;
        if (a.gate_partial != nullptr)
          a.gate_partial[(int64_t)unit * C + c] = fmaf(param_at(a.pw, 1.f, c), sa, param_at(a.pb, 0.f, c) * sb);
        if (mine != nullptr) {
          const float g = param_at(gate, 1.f, c);
          mine[c] = fmaf(g, sa, first ? 0.f : mine[c]);
          mine[C + c] = fmaf(g, sb, first ? 0.f : mine[C + c]);
        }
      });
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) acc_a[k][j] = acc_b[k][j] = 0.f;
    }
  }
  if (mine != nullptr)
    flush(acc_nw, acc_nb, [&](int c, float sw, float sb) {
      mine[2 * C + c] = sw;
      mine[3 * C + c] = sb;
    });
}

template <int DTH, int DTX, int kG, int kK, bool kVec, int kF>
void launch_bwd(const TailArgs& a, const TailBwdPlan& p, hipStream_t s) {
  if constexpr (kVec || kK < 3)  // tail_bwd_most
    tail_bwd_kernel<DTH, DTX, kG, kK, kVec, kF><<<p.blocks, tail_threads(kG), 0, s>>>(a);
}

template <int DTH, int DTX>
void dispatch_bwd(const TailArgs& a, const TailBwdPlan& p, bool vec, hipStream_t s) {
  TERRA_TAIL_SHAPES(launch_bwd, p.shape, (DTX == TERRA_DTYPE_F32 ? 2 : 3), a.flags, vec, a, p, s)
}

}  // namespace
}  // namespace terra
