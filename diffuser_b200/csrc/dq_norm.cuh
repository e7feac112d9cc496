// dq_norm.cuh -- the boundary between two DiT blocks in one pass, forward and
// backward (dq_gated_norm, include/dq_dit.h).
//
//   s = x + rs * gate * Npost(y) * wpost      h = Npre(s) * wpre * (1 + scale) + shift
//
// Bound: HBM.  Forward 8 bytes per element (x, y in; s, h out), backward 12
// (ds, dh, s, y in; dx, dy out), against a few tens of instructions.  A CTA
// takes one token row at a time, every feature in registers (thread i owns
// 4-feature runs i, i + threads, ...), and walks rows with the next row's
// operands already loading while the sums of this one go around: the block
// reductions' latency then costs nothing as long as two or more CTAs share an
// SM.  Each reduction has its own shared words, doubled by row parity, so it
// takes one barrier.
//
// Backward.  With t = Npre(s), m = wpre (1 + scale), dt = dh m, and yh = Npost(y):
//   dx = ds + rstd_s (dt - [mean dt] - t mean(dt t))            (mean dt: LayerNorm only)
//   dq = rs gate wpost dx,  dy = rstd_y (dq - [mean dq] - yh mean(dq yh))
// and the sums over tokens need only three per-column accumulators,
//   q0 = sum dh,  q1 = sum dh t,  q2 = sum dx yh,
// because dshift = q0, dscale = wpre q1, dgate = rs wpost q2 per batch element
// and dwpre = sum_b (1 + scale_b) q1_b, dwpost = rs sum_b gate_b q2_b.  A CTA
// keeps them in registers over its run of rows of one batch element and writes
// them once; a second kernel adds the runs in order (no atomics).
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

namespace dq {

enum : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };

__device__ __forceinline__ void unpack4(uint2 u, float* v) {
  v[0] = __uint_as_float(u.x << 16);
  v[1] = __uint_as_float(u.x & 0xFFFF0000u);
  v[2] = __uint_as_float(u.y << 16);
  v[3] = __uint_as_float(u.y & 0xFFFF0000u);
}
__device__ __forceinline__ uint2 pack4(const float* v) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]);
  const __nv_bfloat162 b = __floats2bfloat162_rn(v[2], v[3]);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// Sum over the CTA's W warps, in the order of block_sum_256 (dq_dit.cuh); red:
// W floats that no other reduction of this row or the next uses.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) t += red[i];
  return t;
}
template <int W>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 t = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    t.x += red[i].x;
    t.y += red[i].y;
  }
  return t;
}

struct NormArgs {
  const __nv_bfloat16 *x, *y, *gate, *scale, *shift, *post_w, *pre_w;
  __nv_bfloat16 *s, *h;
  int64_t ld_x, ld_y, ld_gate, ld_mod, ld_s, ld_h, T;
  int S, D, post, pre;
  float rs, eps;
};

template <bool OPS>
__device__ __forceinline__ float op_round(float v) {
  return OPS ? __bfloat162float(__float2bfloat16_rn(v)) : v;
}

template <int NPT, bool OPS>
__global__ void __launch_bounds__(256) gated_norm_kernel(const NormArgs a) {
  __shared__ float red[2][4][8];
  const int nrun = a.D / 4;
  const float dim = static_cast<float>(a.D);
  uint2 nx[NPT], ny[NPT];
  auto fetch = [&](int64_t t) {
    const uint2* xr = reinterpret_cast<const uint2*>(a.x + t * a.ld_x);
    const uint2* yr = reinterpret_cast<const uint2*>(a.y + t * a.ld_y);
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + 256 * j;
      nx[j] = ny[j] = make_uint2(0u, 0u);
      if (r < nrun) {
        nx[j] = xr[r];
        ny[j] = yr[r];
      }
    }
  };
  fetch(blockIdx.x);
  int par = 0;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x, par ^= 1) {
    float v[NPT][4];
    uint2 cx[NPT];
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      cx[j] = nx[j];
      unpack4(ny[j], v[j]);
    }
    if (t + gridDim.x < a.T) fetch(t + gridDim.x);
    const int64_t b = t / a.S;

    // the norm behind the block
    if (a.post != kNormNone) {
      float mean = 0.f;
      if (a.post == kNormLayer) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NPT; ++j)
          if (threadIdx.x + 256 * j < nrun) sum += (v[j][0] + v[j][1]) + (v[j][2] + v[j][3]);
        mean = row_sum<8>(sum, red[par][0]) / dim;
      }
      float sq = 0.f;
#pragma unroll
      for (int j = 0; j < NPT; ++j)
        if (threadIdx.x + 256 * j < nrun) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float d = v[j][e] - mean;
            sq += d * d;
          }
        }
      const float rstd = rsqrtf(row_sum<8>(sq, red[par][1]) / dim + a.eps);
#pragma unroll
      for (int j = 0; j < NPT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>((v[j][e] - mean) * rstd);
    }
    // weight, gate, residual scale, residual
    const uint2* pw = reinterpret_cast<const uint2*>(a.post_w);
    const uint2* gt = reinterpret_cast<const uint2*>(a.gate + b * a.ld_gate);
    uint2* so = reinterpret_cast<uint2*>(a.s + t * a.ld_s);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + 256 * j;
      if (r < nrun) {
        float c[4];
        if (a.post_w != nullptr) {
          unpack4(__ldg(pw + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>(v[j][e] * c[e]);
        }
        if (a.gate != nullptr) {
          unpack4(__ldg(gt + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>(c[e] * v[j][e]);
        }
        if (a.rs != 1.0f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>(a.rs * v[j][e]);
        }
        unpack4(cx[j], c);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = c[e] + v[j][e];
        const uint2 u = pack4(v[j]);
        so[r] = u;
        unpack4(u, v[j]);  // the next norm sees s as stored
        sum += (v[j][0] + v[j][1]) + (v[j][2] + v[j][3]);
      }
    }
    // the norm before the next block
    float mean = 0.f;
    if (a.pre == kNormLayer) mean = row_sum<8>(sum, red[par][2]) / dim;
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < NPT; ++j)
      if (threadIdx.x + 256 * j < nrun) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float d = v[j][e] - mean;
          sq += d * d;
        }
      }
    const float rstd = rsqrtf(row_sum<8>(sq, red[par][3]) / dim + a.eps);
    const uint2* qw = reinterpret_cast<const uint2*>(a.pre_w);
    const uint2* sc = reinterpret_cast<const uint2*>(a.scale + b * a.ld_mod);
    const uint2* sh = reinterpret_cast<const uint2*>(a.shift + b * a.ld_mod);
    uint2* ho = reinterpret_cast<uint2*>(a.h + t * a.ld_h);
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + 256 * j;
      if (r < nrun) {
        float c[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>((v[j][e] - mean) * rstd);
        if (a.pre_w != nullptr) {
          unpack4(__ldg(qw + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>(v[j][e] * c[e]);
        }
        if (a.scale != nullptr) {
          unpack4(__ldg(sc + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = op_round<OPS>(v[j][e] * op_round<OPS>(c[e] + 1.0f));
        }
        if (a.shift != nullptr) {
          unpack4(__ldg(sh + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = v[j][e] + c[e];
        }
        ho[r] = pack4(v[j]);
      }
    }
  }
}

struct NormGradArgs {
  const __nv_bfloat16 *ds, *dh, *s, *y, *gate, *scale, *post_w, *pre_w;
  __nv_bfloat16 *dx, *dy;
  float* part;  // [B, chunks, 3, D]
  int64_t ld_ds, ld_dh, ld_s, ld_y, ld_gate, ld_mod, ld_dx, ld_dy;
  int S, D, post, pre, rows_per_chunk;
  float rs, eps;
};

// CTA (chunk, batch element): rows chunk * rows_per_chunk .. of one element.
template <int THREADS, int NPT>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1)
    gated_norm_backward_kernel(const NormGradArgs a) {
  constexpr int W = THREADS / 32;
  __shared__ float2 red[2][4][W];
  const int nrun = a.D / 4;
  const float inv = 1.0f / static_cast<float>(a.D);
  const int64_t b = blockIdx.y;
  const int r_lo = blockIdx.x * a.rows_per_chunk, r_hi = min(a.S, r_lo + a.rows_per_chunk);
  const uint2* gt = reinterpret_cast<const uint2*>(a.gate + b * a.ld_gate);
  const uint2* sc = reinterpret_cast<const uint2*>(a.scale + b * a.ld_mod);
  const uint2* pw = reinterpret_cast<const uint2*>(a.post_w);
  const uint2* qw = reinterpret_cast<const uint2*>(a.pre_w);
  float q0[NPT][4] = {}, q1[NPT][4] = {}, q2[NPT][4] = {};
  uint2 n_ds[NPT], n_dh[NPT], n_s[NPT], n_y[NPT];
  auto fetch = [&](int row) {
    const int64_t t = b * a.S + row;
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + THREADS * j;
      n_ds[j] = n_dh[j] = n_s[j] = n_y[j] = make_uint2(0u, 0u);
      if (r < nrun) {
        n_s[j] = reinterpret_cast<const uint2*>(a.s + t * a.ld_s)[r];
        n_y[j] = reinterpret_cast<const uint2*>(a.y + t * a.ld_y)[r];
        n_dh[j] = reinterpret_cast<const uint2*>(a.dh + t * a.ld_dh)[r];
        if (a.ds != nullptr) n_ds[j] = reinterpret_cast<const uint2*>(a.ds + t * a.ld_ds)[r];
      }
    }
  };
  if (r_lo < r_hi) fetch(r_lo);
  int par = 0;
  for (int row = r_lo; row < r_hi; ++row, par ^= 1) {
    const int64_t t = b * a.S + row;
    uint2 u_ds[NPT], u_dh[NPT], u_s[NPT], u_y[NPT];
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      u_ds[j] = n_ds[j];
      u_dh[j] = n_dh[j];
      u_s[j] = n_s[j];
      u_y[j] = n_y[j];
    }
    if (row + 1 < r_hi) fetch(row + 1);
    // statistics of s (x) and y (y); idle threads hold zeros
    float2 mean = make_float2(0.f, 0.f);
    if (a.pre == kNormLayer || a.post == kNormLayer) {
      float2 sum = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        float p[4], q[4];
        unpack4(u_s[j], p);
        unpack4(u_y[j], q);
        sum.x += (p[0] + p[1]) + (p[2] + p[3]);
        sum.y += (q[0] + q[1]) + (q[2] + q[3]);
      }
      sum = row_sum2<W>(sum, red[par][0]);
      if (a.pre == kNormLayer) mean.x = sum.x * inv;
      if (a.post == kNormLayer) mean.y = sum.y * inv;
    }
    float2 sq = make_float2(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < NPT; ++j)
      if (threadIdx.x + THREADS * j < nrun) {
        float p[4], q[4];
        unpack4(u_s[j], p);
        unpack4(u_y[j], q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sq.x += (p[e] - mean.x) * (p[e] - mean.x);
          sq.y += (q[e] - mean.y) * (q[e] - mean.y);
        }
      }
    sq = row_sum2<W>(sq, red[par][1]);
    const float rstd_s = rsqrtf(sq.x * inv + a.eps);
    const float rstd_y = a.post == kNormNone ? 1.0f : rsqrtf(sq.y * inv + a.eps);

    // dt = dh wpre (1 + scale); q0, q1
    float dt[NPT][4];
    float2 d = make_float2(0.f, 0.f);  // sum dt, sum dt t
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + THREADS * j;
      if (r < nrun) {
        float s4[4], c[4];
        unpack4(u_s[j], s4);
        unpack4(u_dh[j], dt[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s4[e] = (s4[e] - mean.x) * rstd_s;
          q0[j][e] += dt[j][e];
          q1[j][e] += dt[j][e] * s4[e];
        }
        if (a.pre_w != nullptr) {
          unpack4(__ldg(qw + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dt[j][e] *= c[e];
        }
        if (a.scale != nullptr) {
          unpack4(__ldg(sc + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dt[j][e] *= 1.0f + c[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          d.x += dt[j][e];
          d.y += dt[j][e] * s4[e];
        }
      }
    }
    d = row_sum2<W>(d, red[par][2]);
    d.x = a.pre == kNormLayer ? d.x * inv : 0.f;
    d.y *= inv;

    // dx, then dq = rs gate wpost dx; q2
    uint2* dxo = reinterpret_cast<uint2*>(a.dx + t * a.ld_dx);
    float2 g = make_float2(0.f, 0.f);  // sum dq, sum dq yh
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + THREADS * j;
      if (r < nrun) {
        float p[4], c[4];
        unpack4(u_s[j], p);
        unpack4(u_ds[j], c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          dt[j][e] = c[e] + rstd_s * (dt[j][e] - d.x - (p[e] - mean.x) * rstd_s * d.y);
        dxo[r] = pack4(dt[j]);
        unpack4(u_y[j], p);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          p[e] = (p[e] - mean.y) * rstd_y;
          q2[j][e] += dt[j][e] * p[e];
        }
        if (a.post_w != nullptr) {
          unpack4(__ldg(pw + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dt[j][e] *= c[e];
        }
        if (a.gate != nullptr) {
          unpack4(__ldg(gt + r), c);
#pragma unroll
          for (int e = 0; e < 4; ++e) dt[j][e] *= c[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dt[j][e] *= a.rs;
          g.x += dt[j][e];
          g.y += dt[j][e] * p[e];
        }
      }
    }
    if (a.post != kNormNone) {
      g = row_sum2<W>(g, red[par][3]);
      g.x = a.post == kNormLayer ? g.x * inv : 0.f;
      g.y *= inv;
    } else {
      g = make_float2(0.f, 0.f);
    }
    uint2* dyo = reinterpret_cast<uint2*>(a.dy + t * a.ld_dy);
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + THREADS * j;
      if (r < nrun) {
        float p[4];
        unpack4(u_y[j], p);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          dt[j][e] = rstd_y * (dt[j][e] - g.x - (p[e] - mean.y) * rstd_y * g.y);
        dyo[r] = pack4(dt[j]);
      }
    }
  }
  float4* part = reinterpret_cast<float4*>(a.part + (b * gridDim.x + blockIdx.x) * 3 * a.D);
#pragma unroll
  for (int j = 0; j < NPT; ++j) {
    const int r = threadIdx.x + THREADS * j;
    if (r < nrun) {
      part[r] = make_float4(q0[j][0], q0[j][1], q0[j][2], q0[j][3]);
      part[nrun + r] = make_float4(q1[j][0], q1[j][1], q1[j][2], q1[j][3]);
      part[2 * nrun + r] = make_float4(q2[j][0], q2[j][1], q2[j][2], q2[j][3]);
    }
  }
}

struct NormReduceArgs {
  const float* part;
  const __nv_bfloat16 *gate, *scale, *post_w, *pre_w;
  float *dgate, *dscale, *dshift, *dpost_w, *dpre_w;
  int64_t ld_gate, ld_mod;
  int B, chunks, D;
  float rs;
};

// CTA: 32 columns.  With eight or more runs per batch element warp w adds every
// 8th of them and the warps' sums meet in order; with fewer, warp w takes every
// 8th batch element whole (a gate per token has as many elements as tokens).
__global__ void __launch_bounds__(256) gated_norm_reduce_kernel(const NormReduceArgs a) {
  __shared__ float red[8][3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const bool in = col < a.D;
  const float wq = in && a.pre_w != nullptr ? __bfloat162float(a.pre_w[col]) : 1.0f;
  const float wp = in && a.post_w != nullptr ? __bfloat162float(a.post_w[col]) : 1.0f;
  float dpre = 0.f, dpost = 0.f;
  auto add = [&](int b, int first, int step, float* q) {
    if (!in) return;
#pragma unroll 4
    for (int c = first; c < a.chunks; c += step) {
      const float* p = a.part + (static_cast<int64_t>(b) * a.chunks + c) * 3 * a.D + col;
#pragma unroll
      for (int i = 0; i < 3; ++i) q[i] += p[static_cast<int64_t>(i) * a.D];
    }
  };
  auto finish = [&](int b, const float* s) {
    if (!in) return;
    const int64_t o = static_cast<int64_t>(b) * a.D + col;
    if (a.dshift != nullptr) a.dshift[o] = s[0];
    if (a.dscale != nullptr) a.dscale[o] = wq * s[1];
    if (a.dgate != nullptr) a.dgate[o] = a.rs * wp * s[2];
    dpre += (a.scale != nullptr ? 1.0f + __bfloat162float(a.scale[b * a.ld_mod + col]) : 1.0f) * s[1];
    dpost += (a.gate != nullptr ? __bfloat162float(a.gate[b * a.ld_gate + col]) : 1.0f) * s[2];
  };
  if (a.chunks < 8) {
    for (int b = warp; b < a.B; b += 8) {
      float q[3] = {};
      add(b, 0, 1, q);
      finish(b, q);
    }
    red[warp][0][lane] = dpre;
    red[warp][1][lane] = dpost;
    __syncthreads();
    dpre = dpost = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      dpre += red[w][0][lane];
      dpost += red[w][1][lane];
    }
  } else {
    for (int b = 0; b < a.B; ++b) {
      float q[3] = {};
      add(b, warp, 8, q);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 3; ++i) red[warp][i][lane] = q[i];
      __syncthreads();
      if (warp == 0) {
        float s[3] = {};
#pragma unroll
        for (int w = 0; w < 8; ++w)
#pragma unroll
          for (int i = 0; i < 3; ++i) s[i] += red[w][i][lane];
        finish(b, s);
      }
    }
  }
  if (warp == 0 && in) {
    if (a.dpre_w != nullptr) a.dpre_w[col] = dpre;
    if (a.dpost_w != nullptr) a.dpost_w[col] = a.rs * dpost;
  }
}

}  // namespace dq
