// dq_norm.cuh -- the boundary between two DiT blocks in one pass, forward and
// backward (dq_gated_norm, include/dq_dit.h).
//
//   s = x + rs * gate * Npost(y) * wpost      h = Npre(s) * wpre * (1 + scale) + shift
//
// Bound: HBM.  Forward 8 bytes per element (x, y in; s, h out), backward 12
// (ds, dh, s, y in; dx, dy out).  At those rates an SM has about 20 and 30
// issue slots per element, so the arithmetic runs on packed float32 pairs
// (fma.rn.f32x2 and its kin) and everything that does not change along a CTA's
// rows is prepared once: a CTA walks rows of one batch element, its factors
// (rs gate wpost; wpre (1 + scale); shift) in shared memory as float32.  One
// row at a time, thread i owning the 4-feature runs i, i + threads, ...; the
// next rows' operands arrive by cp.async in slots that only their own thread
// reads (no barrier).  Each block reduction has shared words of its own,
// doubled by row parity, so it takes one barrier.  (With scalar arithmetic,
// bf16 factors from L1 and the next row prefetched in registers: 42 instructions
// per element and 35 us forward, 68 and 98 us backward at 4608 x 4096, where
// forward now takes 26.5, 5.7 TB/s, and backward with its reduction 52.)  The
// backward kernel is bound by latency: 255 registers and 96 KB leave two CTAs,
// eight warps, per SM, whose issue slots are 33% busy and DRAM 4.4 TB/s; they
// stall on shared-memory reads, fixed latencies, loads, the row's barriers.
//
// Backward.  With t = Npre(s), m = wpre (1 + scale), dt = dh m, and yh = Npost(y):
//   dx = ds + rstd_s (dt - [mean dt] - t mean(dt t))            (mean dt: LayerNorm only)
//   dq = rs gate wpost dx,  dy = rstd_y (dq - [mean dq] - yh mean(dq yh))
// and the sums over tokens need only three per-column accumulators,
//   q0 = sum dh,  q1 = sum dh t,  q2 = sum dx yh,
// because dshift = q0, dscale = wpre q1, dgate = rs wpost q2 per batch element
// and dwpre = sum_b (1 + scale_b) q1_b, dwpost = rs sum_b gate_b q2_b.  A CTA
// keeps them in registers over its rows and writes them once; a second kernel
// adds the CTAs' in order (no atomics).
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "dq_f32x2.cuh"
#include "dq_ptx.cuh"
#include "dq_tile.cuh"

namespace dq {

enum : int { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };

// Thread-private 8-byte copy into shared memory.
__device__ __forceinline__ void cp_async_8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// Sum over the CTA's 8 warps, in the order of block_sum_256 (dq_dit.cuh); red:
// 8 floats (16-byte aligned) that no other reduction of this row or the next uses.
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  const float4 a = *reinterpret_cast<const float4*>(red), b = *reinterpret_cast<const float4*>(red + 4);
  float t = 0.f;
  t += a.x;
  t += a.y;
  t += a.z;
  t += a.w;
  t += b.x;
  t += b.y;
  t += b.z;
  t += b.w;
  return t;
}
// Two sums at once over W warps; red: W pairs (16-byte aligned).
template <int W>
__device__ __forceinline__ float2 row_sum2(F2 v, float2* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float2 u = unpair(v);
    v = add2(v, f2(__shfl_xor_sync(0xffffffffu, u.x, o), __shfl_xor_sync(0xffffffffu, u.y, o)));
  }
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = unpair(v);
  __syncthreads();
  F2 t = f2(0.f);
#pragma unroll
  for (int i = 0; i < W / 2; ++i) {
    const float4 u = *reinterpret_cast<const float4*>(red + 2 * i);
    t = add2(t, add2(f2(u.x, u.y), f2(u.z, u.w)));
  }
  return unpair(t);
}

struct NormArgs {
  const __nv_bfloat16 *x, *y, *gate, *scale, *shift, *post_w, *pre_w;
  __nv_bfloat16 *s, *h;
  int64_t ld_x, ld_y, ld_gate, ld_mod, ld_s, ld_h;
  int S, D, post, pre, chunks;
  float rs, eps;
};

// This thread's run r of the three factor rows of batch element b, float32:
// rs gate wpost, wpre (1 + scale), shift.
struct NormFactors {
  const uint2 *gate, *scale, *shift, *post_w, *pre_w;
  float rs;
  __device__ __forceinline__ static void times(float* m, const uint2* p, int r, float plus) {
    if (p == nullptr) return;
    const uint2 u = __ldg(p + r);
    m[0] *= __uint_as_float(u.x << 16) + plus;
    m[1] *= __uint_as_float(u.x & 0xFFFF0000u) + plus;
    m[2] *= __uint_as_float(u.y << 16) + plus;
    m[3] *= __uint_as_float(u.y & 0xFFFF0000u) + plus;
  }
  __device__ __forceinline__ float4 behind(int r) const {
    float m[4] = {rs, rs, rs, rs};
    times(m, post_w, r, 0.f);
    times(m, gate, r, 0.f);
    return make_float4(m[0], m[1], m[2], m[3]);
  }
  __device__ __forceinline__ float4 before(int r) const {
    float m[4] = {1.f, 1.f, 1.f, 1.f};
    times(m, pre_w, r, 0.f);
    times(m, scale, r, 1.f);
    return make_float4(m[0], m[1], m[2], m[3]);
  }
  __device__ __forceinline__ float4 shifts(int r) const {
    float m[4] = {1.f, 1.f, 1.f, 1.f};
    if (shift == nullptr) return make_float4(0.f, 0.f, 0.f, 0.f);
    times(m, shift, r, 0.f);
    return make_float4(m[0], m[1], m[2], m[3]);
  }
};

__device__ __forceinline__ F2 bf16_round2(F2 a) { return widen(narrow(a)); }

// CTA (batch element, chunk): rows chunk, chunk + chunks, ... of the element.
// OPS rounds after every op of the tensor chain, from the bf16 factors, with
// the sums in the order of adaln_modulate_kernel: the same bits.
constexpr int kNormThreads = 256;
constexpr int kNormAhead = 2;  // rows whose operands are on their way
// FULL: D is NPT runs for every thread.
template <int NPT, bool OPS, bool FULL>
__global__ void __launch_bounds__(kNormThreads, NPT <= 4 ? 3 : 2) gated_norm_kernel(const NormArgs a) {
  __shared__ __align__(16) float red[2][4][8];
  extern __shared__ __align__(16) uint8_t smem[];
  const int nrun = a.D / 4;
  const float dim = static_cast<float>(a.D), inv = 1.0f / dim;
  auto mean_of = [&](float sum) { return OPS ? sum / dim : sum * inv; };
  const int64_t b = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x - static_cast<int>(b) * a.chunks;
  const NormFactors f = {reinterpret_cast<const uint2*>(a.gate == nullptr ? nullptr : a.gate + b * a.ld_gate),
                         reinterpret_cast<const uint2*>(a.scale == nullptr ? nullptr : a.scale + b * a.ld_mod),
                         reinterpret_cast<const uint2*>(a.shift == nullptr ? nullptr : a.shift + b * a.ld_mod),
                         reinterpret_cast<const uint2*>(a.post_w), reinterpret_cast<const uint2*>(a.pre_w), a.rs};
  // slots [row][x, y][run], then (not OPS) the factor rows
  const uint32_t slot0 = smem_u32(smem) + 8u * threadIdx.x;
  const uint32_t row_bytes = 8u * static_cast<uint32_t>(nrun);
  float4* fac = reinterpret_cast<float4*>(smem + kNormAhead * 2 * row_bytes);
  auto fetch = [&](int row, int slot) {
    if (row < a.S) {
      const int64_t t = b * a.S + row;
      const uint2* xr = reinterpret_cast<const uint2*>(a.x + t * a.ld_x);
      const uint2* yr = reinterpret_cast<const uint2*>(a.y + t * a.ld_y);
      const uint32_t dst = slot0 + static_cast<uint32_t>(slot) * 2u * row_bytes;
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        const int r = threadIdx.x + kNormThreads * j;
        if (FULL || r < nrun) {
          cp_async_8(dst + 8u * kNormThreads * j, xr + r);
          cp_async_8(dst + row_bytes + 8u * kNormThreads * j, yr + r);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kNormAhead; ++i) fetch(chunk + i * a.chunks, i);
  if constexpr (!OPS) {
#pragma unroll
    for (int j = 0; j < NPT; ++j) {  // each thread reads back what it wrote
      const int r = threadIdx.x + kNormThreads * j;
      if (FULL || r < nrun) {
        fac[r] = f.behind(r);
        fac[nrun + r] = f.before(r);
        fac[2 * nrun + r] = f.shifts(r);
      }
    }
  }
  int par = 0, slot = 0;
  for (int row = chunk; row < a.S; row += a.chunks, par ^= 1, slot = slot + 1 == kNormAhead ? 0 : slot + 1) {
    const int64_t t = b * a.S + row;
    cp_async_wait<kNormAhead - 1>();
    const uint32_t src = slot0 + static_cast<uint32_t>(slot) * 2u * row_bytes;
    F2 v[NPT][2];
    uint2 cx[NPT];
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + kNormThreads * j;
      cx[j] = make_uint2(0u, 0u);
      uint2 y = make_uint2(0u, 0u);
      if (FULL || r < nrun) {
        cx[j] = lds64(src + 8u * kNormThreads * j);
        y = lds64(src + row_bytes + 8u * kNormThreads * j);
      }
      v[j][0] = widen(y.x);
      v[j][1] = widen(y.y);
    }
    fetch(row + kNormAhead * a.chunks, slot);

    // (v - mean) squared, summed: in adaln_modulate_kernel's order with OPS
    auto squares = [&](float mean) {
      if constexpr (OPS) {
        float sq = 0.f;
#pragma unroll
        for (int j = 0; j < NPT; ++j)
          if (FULL || threadIdx.x + kNormThreads * j < nrun) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              const float2 u = unpair(v[j][p]);
              const float d0 = u.x - mean, d1 = u.y - mean;
              sq += d0 * d0;
              sq += d1 * d1;
            }
          }
        return sq;
      } else {
        F2 sq = f2(0.f);
        const F2 m = f2(-mean);
#pragma unroll
        for (int j = 0; j < NPT; ++j)
          if (FULL || threadIdx.x + kNormThreads * j < nrun) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              const F2 d = add2(v[j][p], m);
              sq = fma2(d, d, sq);
            }
          }
        return sum_pair(sq);
      }
    };
    auto sums = [&]() {  // idle runs hold zeros
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NPT; ++j) sum += sum_pair(v[j][0]) + sum_pair(v[j][1]);
      return sum;
    };

    // the norm behind the block
    if (a.post != kNormNone) {
      const float mean = a.post == kNormLayer ? mean_of(row_sum(sums(), red[par][0])) : 0.f;
      const float rstd = rsqrtf(mean_of(row_sum(squares(mean), red[par][1])) + a.eps);
#pragma unroll
      for (int j = 0; j < NPT; ++j)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          v[j][p] = mul2(add2(v[j][p], f2(-mean)), f2(rstd));
          if constexpr (OPS) v[j][p] = bf16_round2(v[j][p]);
        }
    }
    // weight, gate, residual scale, residual
    uint2* so = reinterpret_cast<uint2*>(a.s + t * a.ld_s);
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + kNormThreads * j;
      if (FULL || r < nrun) {
        uint2 u;
        if constexpr (OPS) {
          if (a.post_w != nullptr) {
            const uint2 c = __ldg(f.post_w + r);
            v[j][0] = bf16_round2(mul2(v[j][0], widen(c.x)));
            v[j][1] = bf16_round2(mul2(v[j][1], widen(c.y)));
          }
          if (a.gate != nullptr) {
            const uint2 c = __ldg(f.gate + r);
            v[j][0] = bf16_round2(mul2(widen(c.x), v[j][0]));
            v[j][1] = bf16_round2(mul2(widen(c.y), v[j][1]));
          }
          if (a.rs != 1.0f) {
            v[j][0] = bf16_round2(mul2(f2(a.rs), v[j][0]));
            v[j][1] = bf16_round2(mul2(f2(a.rs), v[j][1]));
          }
          u = make_uint2(narrow(add2(widen(cx[j].x), v[j][0])), narrow(add2(widen(cx[j].y), v[j][1])));
        } else {
          const float4 g = fac[r];
          u = make_uint2(narrow(fma2(v[j][0], f2(g.x, g.y), widen(cx[j].x))),
                         narrow(fma2(v[j][1], f2(g.z, g.w), widen(cx[j].y))));
        }
        so[r] = u;
        v[j][0] = widen(u.x);  // the next norm sees s as stored
        v[j][1] = widen(u.y);
      } else {
        v[j][0] = v[j][1] = f2(0.f);
      }
    }
    // the norm before the next block
    const float mean = a.pre == kNormLayer ? mean_of(row_sum(sums(), red[par][2])) : 0.f;
    const float rstd = rsqrtf(mean_of(row_sum(squares(mean), red[par][3])) + a.eps);
    uint2* ho = reinterpret_cast<uint2*>(a.h + t * a.ld_h);
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + kNormThreads * j;
      if (FULL || r < nrun) {
        F2 n0 = mul2(add2(v[j][0], f2(-mean)), f2(rstd)), n1 = mul2(add2(v[j][1], f2(-mean)), f2(rstd));
        if constexpr (OPS) {
          n0 = bf16_round2(n0);
          n1 = bf16_round2(n1);
          if (a.pre_w != nullptr) {
            const uint2 c = __ldg(f.pre_w + r);
            n0 = bf16_round2(mul2(n0, widen(c.x)));
            n1 = bf16_round2(mul2(n1, widen(c.y)));
          }
          if (a.scale != nullptr) {
            const uint2 c = __ldg(f.scale + r);
            n0 = bf16_round2(mul2(n0, bf16_round2(add2(widen(c.x), f2(1.0f)))));
            n1 = bf16_round2(mul2(n1, bf16_round2(add2(widen(c.y), f2(1.0f)))));
          }
          if (a.shift != nullptr) {
            const uint2 c = __ldg(f.shift + r);
            n0 = add2(n0, widen(c.x));
            n1 = add2(n1, widen(c.y));
          }
        } else {
          const float4 m = fac[nrun + r], h = fac[2 * nrun + r];
          n0 = fma2(n0, f2(m.x, m.y), f2(h.x, h.y));
          n1 = fma2(n1, f2(m.z, m.w), f2(h.z, h.w));
        }
        ho[r] = make_uint2(narrow(n0), narrow(n1));
      }
    }
  }
  cp_async_wait<0>();
}

struct NormGradArgs {
  const __nv_bfloat16 *ds, *dh, *s, *y, *gate, *scale, *post_w, *pre_w;
  __nv_bfloat16 *dx, *dy;
  float* part;  // [B, chunks, 3, D]
  int64_t ld_ds, ld_dh, ld_s, ld_y, ld_gate, ld_mod, ld_dx, ld_dy;
  int S, D, post, pre, chunks;
  float rs, eps;
};

// CTA (batch element, chunk): rows chunk, chunk + chunks, ... of the element.
// Few threads with many features each: a row's reductions and addresses cost
// every warp the same whatever it owns (4608 x 4096: 63 us with 16 warps per
// row, 49 with 8, 46 with 4).
constexpr int kNormGradAhead = 2;
__host__ __device__ constexpr int norm_grad_ctas(int threads, int npt) { return threads > 128 ? 1 : npt <= 4 ? 4 : 2; }
template <int THREADS, int NPT, bool FULL>
__global__ void __launch_bounds__(THREADS, norm_grad_ctas(THREADS, NPT))
    gated_norm_backward_kernel(const NormGradArgs a) {
  constexpr int W = THREADS / 32;
  __shared__ __align__(16) float2 red[2][4][W];
  extern __shared__ __align__(16) uint8_t smem[];
  const int nrun = a.D / 4;
  const float inv = 1.0f / static_cast<float>(a.D);
  const int64_t b = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x - static_cast<int>(b) * a.chunks;
  const uint32_t slot0 = smem_u32(smem) + 8u * threadIdx.x;
  const uint32_t row_bytes = 8u * static_cast<uint32_t>(nrun);
  // slots [row][s, y, dh, ds][run], then the factor rows
  float4* fac = reinterpret_cast<float4*>(smem + kNormGradAhead * 4 * row_bytes);
  auto fetch = [&](int row, int slot) {
    if (row < a.S) {
      const int64_t t = b * a.S + row;
      const uint32_t dst = slot0 + static_cast<uint32_t>(slot) * 4u * row_bytes;
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        const int r = threadIdx.x + THREADS * j;
        if (FULL || r < nrun) {
          const uint32_t d = dst + 8u * THREADS * j;
          cp_async_8(d, reinterpret_cast<const uint2*>(a.s + t * a.ld_s) + r);
          cp_async_8(d + row_bytes, reinterpret_cast<const uint2*>(a.y + t * a.ld_y) + r);
          cp_async_8(d + 2 * row_bytes, reinterpret_cast<const uint2*>(a.dh + t * a.ld_dh) + r);
        }
      }
      if (a.ds != nullptr) {
#pragma unroll
        for (int j = 0; j < NPT; ++j) {
          const int r = threadIdx.x + THREADS * j;
          if (FULL || r < nrun)
            cp_async_8(dst + 3 * row_bytes + 8u * THREADS * j, reinterpret_cast<const uint2*>(a.ds + t * a.ld_ds) + r);
        }
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kNormGradAhead; ++i) fetch(chunk + i * a.chunks, i);
  const NormFactors f = {reinterpret_cast<const uint2*>(a.gate == nullptr ? nullptr : a.gate + b * a.ld_gate),
                         reinterpret_cast<const uint2*>(a.scale == nullptr ? nullptr : a.scale + b * a.ld_mod),
                         nullptr, reinterpret_cast<const uint2*>(a.post_w), reinterpret_cast<const uint2*>(a.pre_w),
                         a.rs};
#pragma unroll
  for (int j = 0; j < NPT; ++j) {  // each thread reads back what it wrote
    const int r = threadIdx.x + THREADS * j;
    if (FULL || r < nrun) {
      fac[r] = f.behind(r);
      fac[nrun + r] = f.before(r);
      if (a.ds == nullptr)  // its slots stay zero
        for (int i = 0; i < kNormGradAhead; ++i)
          *reinterpret_cast<uint2*>(smem + (4 * i + 3) * row_bytes + 8 * r) = make_uint2(0u, 0u);
    }
  }
  F2 q0[NPT][2], q1[NPT][2], q2[NPT][2];
#pragma unroll
  for (int j = 0; j < NPT; ++j)
#pragma unroll
    for (int p = 0; p < 2; ++p) q0[j][p] = q1[j][p] = q2[j][p] = f2(0.f);
  const bool means = a.pre == kNormLayer || a.post == kNormLayer;
  int par = 0, slot = 0;
  for (int row = chunk; row < a.S; row += a.chunks, par ^= 1, slot = slot + 1 == kNormGradAhead ? 0 : slot + 1) {
    const int64_t t = b * a.S + row;
    cp_async_wait<kNormGradAhead - 1>();
    const uint32_t src = slot0 + static_cast<uint32_t>(slot) * 4u * row_bytes;
    uint2 us[NPT], uy[NPT];
    F2 dt[NPT][2];  // dh
    uint2 ud[NPT];  // ds
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + THREADS * j;
      const uint32_t d = src + 8u * THREADS * j;
      us[j] = uy[j] = ud[j] = make_uint2(0u, 0u);
      uint2 u = make_uint2(0u, 0u);
      if (FULL || r < nrun) {
        us[j] = lds64(d);
        uy[j] = lds64(d + row_bytes);
        u = lds64(d + 2 * row_bytes);
        ud[j] = lds64(d + 3 * row_bytes);
      }
      dt[j][0] = widen(u.x);
      dt[j][1] = widen(u.y);
    }
    fetch(row + kNormGradAhead * a.chunks, slot);
    // statistics of s (x) and y (y); idle runs hold zeros
    float2 mean = make_float2(0.f, 0.f);
    if (means) {
      F2 ms = f2(0.f), my = f2(0.f);
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        ms = add2(ms, add2(widen(us[j].x), widen(us[j].y)));
        my = add2(my, add2(widen(uy[j].x), widen(uy[j].y)));
      }
      const float2 sum = row_sum2<W>(f2(sum_pair(ms), sum_pair(my)), red[par][0]);
      if (a.pre == kNormLayer) mean.x = sum.x * inv;
      if (a.post == kNormLayer) mean.y = sum.y * inv;
    }
    float rstd_s, rstd_y = 1.0f;
    {
      F2 ss = f2(0.f), sy = f2(0.f);
#pragma unroll
      for (int j = 0; j < NPT; ++j)
        if (FULL || threadIdx.x + THREADS * j < nrun) {
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const F2 ds = add2(widen(p ? us[j].y : us[j].x), f2(-mean.x));
            const F2 dy = add2(widen(p ? uy[j].y : uy[j].x), f2(-mean.y));
            ss = fma2(ds, ds, ss);
            sy = fma2(dy, dy, sy);
          }
        }
      const float2 sq = row_sum2<W>(f2(sum_pair(ss), sum_pair(sy)), red[par][1]);
      rstd_s = rsqrtf(sq.x * inv + a.eps);
      if (a.post != kNormNone) rstd_y = rsqrtf(sq.y * inv + a.eps);
    }
    // dt = dh wpre (1 + scale); q0, q1; sums of dt and dt t
    float2 d;
    {
      F2 d0 = f2(0.f), d1 = f2(0.f);
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        const int r = threadIdx.x + THREADS * j;
        if (FULL || r < nrun) {
          const float4 m = fac[nrun + r];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const F2 tt = mul2(add2(widen(p ? us[j].y : us[j].x), f2(-mean.x)), f2(rstd_s));
            q0[j][p] = add2(q0[j][p], dt[j][p]);
            q1[j][p] = fma2(dt[j][p], tt, q1[j][p]);
            dt[j][p] = mul2(dt[j][p], p ? f2(m.z, m.w) : f2(m.x, m.y));
            d0 = add2(d0, dt[j][p]);
            d1 = fma2(dt[j][p], tt, d1);
          }
        }
      }
      d = row_sum2<W>(f2(sum_pair(d0), sum_pair(d1)), red[par][2]);
      d.x = a.pre == kNormLayer ? d.x * inv : 0.f;
      d.y *= inv;
    }
    // dx = ds + rstd (dt - mean dt - t mean(dt t)); q2; dq = rs gate wpost dx
    uint2* dxo = reinterpret_cast<uint2*>(a.dx + t * a.ld_dx);
    float2 g;
    {
      F2 g0 = f2(0.f), g1 = f2(0.f);
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        const int r = threadIdx.x + THREADS * j;
        if (FULL || r < nrun) {
          const float4 n = fac[r];
          uint32_t o[2];
#pragma unroll
          for (int p = 0; p < 2; ++p) {
            const F2 tt = mul2(add2(widen(p ? us[j].y : us[j].x), f2(-mean.x)), f2(rstd_s));
            const F2 in = fma2(tt, f2(-d.y), add2(dt[j][p], f2(-d.x)));
            const F2 dx = fma2(in, f2(rstd_s), widen(p ? ud[j].y : ud[j].x));
            o[p] = narrow(dx);
            const F2 yh = mul2(add2(widen(p ? uy[j].y : uy[j].x), f2(-mean.y)), f2(rstd_y));
            q2[j][p] = fma2(dx, yh, q2[j][p]);
            dt[j][p] = mul2(dx, p ? f2(n.z, n.w) : f2(n.x, n.y));
            g0 = add2(g0, dt[j][p]);
            g1 = fma2(dt[j][p], yh, g1);
          }
          dxo[r] = make_uint2(o[0], o[1]);
        }
      }
      g = make_float2(0.f, 0.f);
      if (a.post != kNormNone) {
        g = row_sum2<W>(f2(sum_pair(g0), sum_pair(g1)), red[par][3]);
        g.x = a.post == kNormLayer ? g.x * inv : 0.f;
        g.y *= inv;
      }
    }
    uint2* dyo = reinterpret_cast<uint2*>(a.dy + t * a.ld_dy);
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
      const int r = threadIdx.x + THREADS * j;
      if (FULL || r < nrun) {
        uint32_t o[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const F2 yh = mul2(add2(widen(p ? uy[j].y : uy[j].x), f2(-mean.y)), f2(rstd_y));
          o[p] = narrow(mul2(fma2(yh, f2(-g.y), add2(dt[j][p], f2(-g.x))), f2(rstd_y)));
        }
        dyo[r] = make_uint2(o[0], o[1]);
      }
    }
  }
  cp_async_wait<0>();
  grid_launch_dependents();
  float4* part = reinterpret_cast<float4*>(a.part + static_cast<int64_t>(blockIdx.x) * 3 * a.D);
#pragma unroll
  for (int j = 0; j < NPT; ++j) {
    const int r = threadIdx.x + THREADS * j;
    if (FULL || r < nrun) {
      auto put = [&](int i, F2 (&q)[2]) {
        const float2 u = unpair(q[0]), w = unpair(q[1]);
        part[i * nrun + r] = make_float4(u.x, u.y, w.x, w.y);
      };
      put(0, q0[j]);
      put(1, q1[j]);
      put(2, q2[j]);
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

// CTA: 32 columns and 32 warps.  With 32 or more chunks per batch element warp w
// adds every 32nd of them (all its loads in flight at once: the sums are latency
// bound, eight warps took 16 us at 2 x 148 chunks x 4096) and the warps' sums
// meet in order; with fewer, warp w takes every 32nd batch element whole (a gate
// per token has as many elements as tokens).
constexpr int kReduceWarps = 32;
__global__ void __launch_bounds__(32 * kReduceWarps) gated_norm_reduce_kernel(const NormReduceArgs a) {
  constexpr int W = kReduceWarps;
  __shared__ float red[W][3][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + lane;
  const bool in = col < a.D;
  const float wq = in && a.pre_w != nullptr ? __bfloat162float(a.pre_w[col]) : 1.0f;
  const float wp = in && a.post_w != nullptr ? __bfloat162float(a.post_w[col]) : 1.0f;
  float dpre = 0.f, dpost = 0.f;
  grid_wait();  // the chunks' sums
  auto add = [&](int b, int first, int step, float* q) {
    if (!in) return;
    for (int c0 = first; c0 < a.chunks; c0 += 8 * step) {
      float u[8][3];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int c = c0 + k * step;
        const float* p = a.part + (static_cast<int64_t>(b) * a.chunks + c) * 3 * a.D + col;
#pragma unroll
        for (int i = 0; i < 3; ++i) u[k][i] = c < a.chunks ? __ldcg(p + static_cast<int64_t>(i) * a.D) : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int i = 0; i < 3; ++i) q[i] += u[k][i];
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
  if (a.chunks < W) {
    for (int b = warp; b < a.B; b += W) {
      float q[3] = {};
      add(b, 0, 1, q);
      finish(b, q);
    }
    red[warp][0][lane] = dpre;
    red[warp][1][lane] = dpost;
    __syncthreads();
    dpre = dpost = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      dpre += red[w][0][lane];
      dpost += red[w][1][lane];
    }
  } else {
    for (int b = 0; b < a.B; ++b) {
      float q[3] = {};
      add(b, warp, W, q);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 3; ++i) red[warp][i][lane] = q[i];
      __syncthreads();
      if (warp == 0) {
        float s[3] = {};
#pragma unroll
        for (int w = 0; w < W; ++w)
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
