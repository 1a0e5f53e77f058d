// Backward of the end of a half-block (residual_norm.h), from the gradients
// of y and z.  No statistic, mask or intermediate of the forward is kept: each
// row is recomputed from h and x in registers, and then
//
//   g  = dz w2,  dY = dy + r2 (g - mean g - yhat mean(g yhat)),  dx = alpha dY
//   dgate += dY m,  dn = keep s gate dY
//   u  = dn w1,  dh = r1 (u - mean u - nhat mean(u nhat))
//   dw2 += dz yhat,  db2 += dz,  dw1 += dn nhat,  db1 += dn
//
// (an RMS norm has no mean g and mean u term; without a norm dY = dy, dh = dn).
// Bound by memory: h, x, dy, dz read once, dh and dx written once.
//
// Sums over rows: a unit is up to slab_rows consecutive rows of one sample,
// workgroups take units in grid strides, and each lane keeps the sums of its
// columns in registers over all of them; the gate's are written out unit by
// unit, since its row changes with the sample.  A second launch adds the
// workgroups' sums (sum_partials_kernel): no atomics, an order that the sizes
// fix.
#include "residual_norm.h"

namespace terra {
namespace {

template <int DTH, int DTX, int kG, int kK, bool kVec>
__global__ __launch_bounds__(tail_threads(kG)) void tail_bwd_kernel(const TailArgs a) {
  constexpr int kThreads = tail_threads(kG), kGroups = kThreads / kG, kCols = kG * kK * kChunkCols;
  constexpr int kHB = ChunkElt<DTH>::kBytes, kXB = ChunkElt<DTX>::kBytes;
  // w1, b1, gate, w2 of the lane's columns: in LDS where several rows share a
  // workgroup, in registers where each lane's columns are its own.
  constexpr bool kLds = kG <= 64;
  __shared__ typename RowSum<kG>::Shared s_red;
  __shared__ __attribute__((aligned(16))) float s_par[kLds ? 4 : 1][kLds ? kCols : 1];
  __shared__ __attribute__((aligned(16))) float s_acc[kGroups > 1 ? kGroups * kCols : 1];
  float r_par[4][kLds ? 1 : kK][kChunkCols];
  const int lane = threadIdx.x % kG, group = threadIdx.x / kG, C = a.C;
  RowSum<kG> sum(&s_red);

  auto stage = [&](int which, const float* p, float none) {
    if constexpr (kLds) {
      for (int c = threadIdx.x; c < kCols; c += kThreads) s_par[which][c] = c >= C ? 0.f : (p == nullptr ? none : p[c]);
    } else {
#pragma unroll
      for (int k = 0; k < kK; ++k) load_params<kVec>(p, none, (lane + kG * k) * kChunkCols, C, r_par[which][k]);
    }
  };
  auto param = [&](int which, int k, float (&f)[kChunkCols]) {
    if constexpr (kLds) {
      const float4* p = reinterpret_cast<const float4*>(&s_par[which][(lane + kG * k) * kChunkCols]);
      const float4 lo = p[0], hi = p[1];
      f[0] = lo.x, f[1] = lo.y, f[2] = lo.z, f[3] = lo.w, f[4] = hi.x, f[5] = hi.y, f[6] = hi.z, f[7] = hi.w;
    } else {
#pragma unroll
      for (int j = 0; j < kChunkCols; ++j) f[j] = r_par[which][k][j];
    }
  };
  stage(0, a.pw, 1.f);
  stage(1, a.pb, 0.f);
  stage(2, a.gate_rows == 1 ? a.gate : nullptr, 1.f);
  stage(3, a.nw, 1.f);
  __syncthreads();
  const uint64_t seed = a.drop.threshold > 0 ? *a.drop.seed : 0;

  float acc_pw[kK][kChunkCols] = {}, acc_pb[kK][kChunkCols] = {}, acc_gate[kK][kChunkCols] = {};
  float acc_nw[kK][kChunkCols] = {}, acc_nb[kK][kChunkCols] = {};
  // The workgroup's sums of one vector: over its row groups, then to dst [C].
  auto flush = [&](float (&acc)[kK][kChunkCols], float* dst) {
    if constexpr (kGroups > 1) {
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) s_acc[group * kCols + (lane + kG * k) * kChunkCols + j] = acc[k][j];
      __syncthreads();
      for (int c = threadIdx.x; c < C; c += kThreads) {
        float t = 0.f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) t += s_acc[g * kCols + c];
        dst[c] = t;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          const int c = (lane + kG * k) * kChunkCols + j;
          if (c < C) dst[c] = acc[k][j];
        }
    }
  };

  for (uint32_t unit = blockIdx.x; unit < a.units; unit += gridDim.x) {
    const uint32_t sample = unit / a.slabs, slab = unit % a.slabs;
    const uint32_t begin = sample * a.per_sample + slab * a.slab_rows;
    const uint32_t end = min(begin + a.slab_rows, (sample + 1) * a.per_sample);
    if (a.gate_rows > 1) {
      __syncthreads();
      stage(2, a.gate + (int64_t)sample * C, 1.f);
      __syncthreads();
    }
    for (uint32_t base = begin; base < end; base += kGroups) {
      const uint32_t row = base + group;
      const bool live = row < end;
      const uint32_t r = live ? row : end - 1;  // a row past the end re-reads the unit's last one
      const int64_t src = a.windows ? a.map.source(r) : (int64_t)r;
      const bool has = src >= 0;
      RowChunk<DTH> hq[kK], dzq[kK];
      RowChunk<DTX> xq[kK], dyq[kK];
      const uint8_t* hp = a.h + (has ? src : 0) * a.h_row_bytes;
      const uint8_t* xp = a.x + (int64_t)r * a.x_row_bytes;
      const uint8_t* dyp = a.dy != nullptr ? a.dy + (int64_t)r * C * kXB : xp;
      const uint8_t* dzp = a.dz != nullptr ? a.dz + (int64_t)r * C * kHB : hp;
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const int col = (lane + kG * k) * kChunkCols;
        const bool in = col < C;
        hq[k] = load_chunk<DTH, kVec>(hp, col, C, in);
        xq[k] = load_chunk<DTX, kVec>(xp, col, C, in);
        dyq[k] = load_chunk<DTX, kVec>(dyp, col, C, in);
        dzq[k] = load_chunk<DTH, kVec>(dzp, col, C, in);
      }
      // The forward: nhat in nv, m, and yhat in yv.
      float nv[kK][kChunkCols], m[kK][kChunkCols], yv[kK][kChunkCols];
      ChunkDraws draws[kK];
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const int col = (lane + kG * k) * kChunkCols;
        unpack<DTH, kVec>(hq[k], nv[k], col, C, has && col < C);
      }
      float r1 = 1.f, r2 = 1.f;
      if (a.post != TERRA_NORM_NONE) r1 = normalise<kG, kK, kVec>(nv, a.post, a.post_eps, a.inv_c, lane, C, sum);
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const int col = (lane + kG * k) * kChunkCols;
        float w[kChunkCols], b[kChunkCols], g[kChunkCols], xv[kChunkCols];
        param(0, k, w);
        param(1, k, b);
        param(2, k, g);
        unpack<DTX, kVec>(xq[k], xv, col, C, col < C);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) m[k][j] = has ? fmaf(nv[k][j], w[j], b[j]) : 0.f;
        if (a.drop.threshold > 0) {
          draws[k] = chunk_draws(seed, (uint32_t)(lane + kG * k), r, a.drop.stream);
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) m[k][j] = kept(draws[k], j, a.drop.threshold) ? m[k][j] * a.drop.scale : 0.f;
        }
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) yv[k][j] = fmaf(a.alpha, xv[j], g[j] * m[k][j]);
      }
      // dY in dv.
      float dv[kK][kChunkCols];
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const int col = (lane + kG * k) * kChunkCols;
        unpack<DTX, kVec>(dyq[k], dv[k], col, C, a.dy != nullptr && col < C);
      }
      if (a.next != TERRA_NORM_NONE && a.dz != nullptr) {
        r2 = normalise<kG, kK, kVec>(yv, a.next, a.next_eps, a.inv_c, lane, C, sum);
        float s0 = 0.f, s1 = 0.f;
        float gv[kK][kChunkCols];
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          const int col = (lane + kG * k) * kChunkCols;
          float w[kChunkCols];
          param(3, k, w);
          unpack<DTH, kVec>(dzq[k], gv[k], col, C, live && col < C);
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) {
            if (live) acc_nw[k][j] = fmaf(gv[k][j], yv[k][j], acc_nw[k][j]);
            acc_nb[k][j] += gv[k][j];
            gv[k][j] *= w[j];
            s0 += gv[k][j];
            s1 = fmaf(gv[k][j], yv[k][j], s1);
          }
        }
        sum.two(s0, s1);
        s0 = a.next == TERRA_NORM_LAYER ? s0 * a.inv_c : 0.f;
        s1 *= a.inv_c;
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) dv[k][j] += r2 * (gv[k][j] - s0 - yv[k][j] * s1);
      }
      // dx, the gate's gradient, and dn in dv.
      const __amdgpu_buffer_rsrc_t dx_out =
          buffer_rsrc(a.dx + (int64_t)base * C * kXB, min(end - base, (uint32_t)kGroups) * (uint32_t)(C * kXB));
#pragma unroll
      for (int k = 0; k < kK; ++k) {
        const int col = (lane + kG * k) * kChunkCols;
        float g[kChunkCols], dxv[kChunkCols];
        param(2, k, g);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) dxv[j] = a.alpha * dv[k][j];
        if (live && col < C) store_chunk<DTX, kVec>(dxv, dx_out, (uint32_t)(group * C + col) * kXB, col, C);
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) {
          if (live && has) acc_gate[k][j] = fmaf(dv[k][j], m[k][j], acc_gate[k][j]);
          dv[k][j] *= g[j];
        }
        if (a.drop.threshold > 0)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j)
            dv[k][j] = kept(draws[k], j, a.drop.threshold) ? dv[k][j] * a.drop.scale : 0.f;
      }
      if (a.post != TERRA_NORM_NONE) {
        float s0 = 0.f, s1 = 0.f;
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          float w[kChunkCols];
          param(0, k, w);
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) {
            if (live && has) {
              acc_pw[k][j] = fmaf(dv[k][j], nv[k][j], acc_pw[k][j]);
              acc_pb[k][j] += dv[k][j];
            }
            dv[k][j] *= w[j];
            s0 += dv[k][j];
            s1 = fmaf(dv[k][j], nv[k][j], s1);
          }
        }
        sum.two(s0, s1);
        s0 = a.post == TERRA_NORM_LAYER ? s0 * a.inv_c : 0.f;
        s1 *= a.inv_c;
#pragma unroll
        for (int k = 0; k < kK; ++k)
#pragma unroll
          for (int j = 0; j < kChunkCols; ++j) dv[k][j] = r1 * (dv[k][j] - s0 - nv[k][j] * s1);
      }
      // In window order each row has a place of its own: a descriptor for it
      // would not be uniform over the wave's rows, so these bounds are the row's.
      if (a.windows) {
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          const int col = (lane + kG * k) * kChunkCols;
          if (live && has && col < C) store_row<DTH, kVec>(dv[k], a.dh + src * C * kHB, col, C);
        }
      } else {
        const __amdgpu_buffer_rsrc_t dh_out =
            buffer_rsrc(a.dh + (int64_t)base * C * kHB, min(end - base, (uint32_t)kGroups) * (uint32_t)(C * kHB));
#pragma unroll
        for (int k = 0; k < kK; ++k) {
          const int col = (lane + kG * k) * kChunkCols;
          if (live && col < C) store_chunk<DTH, kVec>(dv[k], dh_out, (uint32_t)(group * C + col) * kHB, col, C);
        }
      }
    }
    if (a.gate_partial != nullptr) {
      flush(acc_gate, a.gate_partial + (int64_t)unit * C);
#pragma unroll
      for (int k = 0; k < kK; ++k)
#pragma unroll
        for (int j = 0; j < kChunkCols; ++j) acc_gate[k][j] = 0.f;
    }
  }
  if (a.partial != nullptr) {
    float* dst = a.partial + (int64_t)blockIdx.x * 4 * C;
    if (a.post != TERRA_NORM_NONE) {
      flush(acc_pw, dst);
      flush(acc_pb, dst + C);
    }
    if (a.next != TERRA_NORM_NONE) {
      flush(acc_nw, dst + 2 * (int64_t)C);
      flush(acc_nb, dst + 3 * (int64_t)C);
    }
  }
}

template <int DTH, int DTX, int kG, int kK>
void launch(const TailArgs& a, const TailBwdPlan& p, bool vec, hipStream_t s) {
  if (vec) tail_bwd_kernel<DTH, DTX, kG, kK, true><<<p.blocks, tail_threads(kG), 0, s>>>(a);
  else tail_bwd_kernel<DTH, DTX, kG, kK, false><<<p.blocks, tail_threads(kG), 0, s>>>(a);
}

template <int DTH, int DTX>
void dispatch(const TailArgs& a, const TailBwdPlan& p, bool vec, hipStream_t s) {
  switch (p.shape.lanes * 10 + p.shape.chunks) {
    case 161: return launch<DTH, DTX, 16, 1>(a, p, vec, s);
    case 321: return launch<DTH, DTX, 32, 1>(a, p, vec, s);
    case 641: return launch<DTH, DTX, 64, 1>(a, p, vec, s);
    case 642: return launch<DTH, DTX, 64, 2>(a, p, vec, s);
    case 2561: return launch<DTH, DTX, 256, 1>(a, p, vec, s);
    case 2562: return launch<DTH, DTX, 256, 2>(a, p, vec, s);
    default: return launch<DTH, DTX, 512, 2>(a, p, vec, s);
  }
}

}  // namespace

// Workgroups: what fits the 256 compute units at once; slabs of the rows of a
// sample so that every workgroup has a unit, and rows enough for its groups.
TailBwdPlan tail_bwd_plan(uint32_t rows, int C, int gate_rows) {
  TailBwdPlan p;
  p.shape = tail_shape(C);
  const uint32_t groups = (uint32_t)(tail_threads(p.shape.lanes) / p.shape.lanes);
  const uint32_t most = p.shape.lanes > 256 ? 256u : (p.shape.chunks > 1 ? 512u : 1024u);
  const uint32_t samples = gate_rows > 1 ? (uint32_t)gate_rows : 1u, per = rows / samples;
  uint32_t slabs = (most + samples - 1) / samples;
  const uint32_t useful = (per + groups - 1) / groups;
  if (slabs > useful) slabs = useful;
  p.slab_rows = (per + slabs - 1) / slabs;
  p.slab_rows = (p.slab_rows + groups - 1) / groups * groups;
  p.slabs = (per + p.slab_rows - 1) / p.slab_rows;
  p.units = p.slabs * samples;
  p.blocks = p.units < most ? p.units : most;
  return p;
}

int launch_tail_bwd(int h_dtype, int x_dtype, const void* args, const TailBwdPlan& plan, bool vec, hipStream_t s) {
  const TailArgs& a = *static_cast<const TailArgs*>(args);
  if (h_dtype == TERRA_DTYPE_F32) dispatch<TERRA_DTYPE_F32, TERRA_DTYPE_F32>(a, plan, vec, s);
  else if (h_dtype == TERRA_DTYPE_BF16 && x_dtype == TERRA_DTYPE_BF16) dispatch<TERRA_DTYPE_BF16, TERRA_DTYPE_BF16>(a, plan, vec, s);
  else if (h_dtype == TERRA_DTYPE_BF16) dispatch<TERRA_DTYPE_BF16, TERRA_DTYPE_F32>(a, plan, vec, s);
  else if (x_dtype == TERRA_DTYPE_F16) dispatch<TERRA_DTYPE_F16, TERRA_DTYPE_F16>(a, plan, vec, s);
  else dispatch<TERRA_DTYPE_F16, TERRA_DTYPE_F32>(a, plan, vec, s);
  return TERRA_OK;
}

}  // namespace terra
