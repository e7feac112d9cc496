// dq_checkpoint.cuh -- activations kept in 8 bits until the backward pass
// (include/dq_adapter.h).
#pragma once

#include "dq_adapter.cuh"
#include "dq_codec.cuh"
#include "dq_f32x2.cuh"

namespace dq {

constexpr int kCkptRun = 128;  // features per scale

// Row and column of a flat index that advances by a constant stride: one
// division at the start instead of one per step (a 64-bit division per 8
// features was a quarter of the pack kernel's instructions).
struct RowWalk {
  int64_t row, step_rows;
  int col, step_cols, width;
  __device__ __forceinline__ RowWalk(int64_t start, int64_t stride, int width_) : width(width_) {
    row = start / width;
    col = static_cast<int>(start - row * width);
    step_rows = stride / width;
    step_cols = static_cast<int>(stride - step_rows * width);
  }
  __device__ __forceinline__ void next() {
    row += step_rows;
    col += step_cols;
    if (col >= width) {
      col -= width;
      ++row;
    }
  }
};

// Pack: 8 lanes per run of 128 features, 16 features per lane (one 32-byte load
// where the rows are 32-byte aligned: 58 us at 6144 x 16384, two of 16 bytes 60),
// four runs per warp (16 lanes per run spend more on the maximum and the scale:
// 75 us; the next run's load issued ahead, or two runs at a time: 63).
// The maximum is taken over bf16 pairs and keeps NaN, so a run that is not
// finite is seen.  Bound: HBM, 3 bytes per feature, 47 us.  An IEEE division per
// feature made pack 127 us, so the quotient is taken as x (1 / scale), off by at
// most 127 (2^-23 + 2^-24) = 2.3e-5 from the exact one, and divided only where
// that could round to another integer: within 1e-4 of a half.  Adding 1.5 2^23 rounds to an integer (ties to
// even) and leaves it in the low bits, without the special-function unit's
// conversions.
constexpr float kRoundMagic = 12582912.0f;  // 1.5 * 2^23
__device__ __forceinline__ void pack_pair(uint32_t w, float scale, F2 inv, uint32_t& c0, uint32_t& c1) {
  const F2 v = widen(w), t = mul2(v, inv);
  F2 u = add2(t, f2(kRoundMagic));
  const float2 d = unpair(add2(t, f2_neg(add2(u, f2(-kRoundMagic)))));
  float2 r = unpair(u);
  if (fmaxf(fabsf(d.x), fabsf(d.y)) > 0.4999f) {
    const float2 x = unpair(v);
    r.x = __fadd_rn(__fdiv_rn(x.x, scale), kRoundMagic);
    r.y = __fadd_rn(__fdiv_rn(x.y, scale), kRoundMagic);
  }
  c0 = __float_as_uint(r.x);
  c1 = __float_as_uint(r.y);
}

// amax / 127, correctly rounded: the product with the rounded 1 / 127, then one
// residual step in fused arithmetic (Markstein's division); the same as the
// IEEE quotient for every bf16 magnitude of at least 1e-12.
__device__ __forceinline__ float over_127(float amax) {
  constexpr float c = 1.0f / 127.0f;
  const float q = amax * c;
  return fmaf(fmaf(-127.0f, q, amax), c, q);
}

// 32 streamed bytes in one instruction (32-byte aligned).
__device__ __forceinline__ void ld_stream32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p));
}

__device__ __forceinline__ void st_global32(void* p, uint4 a, uint4 b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
               "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

__global__ void __launch_bounds__(256)
    checkpoint_pack_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int64_t M, int nrun, int K,
                           bool wide, int8_t* __restrict__ codes, float* __restrict__ scales) {
  const int sub = threadIdx.x & 7;  // lane of the run's eight
  RowWalk at(blockIdx.x * 32ll + (threadIdx.x >> 3), static_cast<int64_t>(gridDim.x) * 32, nrun);
  while (__any_sync(0xffffffffu, at.row < M)) {
    const int64_t row = at.row;
    const int run = at.col, k = run * kCkptRun + sub * 16;
    const bool in = row < M && k < K;  // K % 16 == 0
    uint4 u[2] = {make_uint4(0u, 0u, 0u, 0u), make_uint4(0u, 0u, 0u, 0u)};
    if (in) {
      const __nv_bfloat16* p = x + row * ldx + k;
      if (wide) {
        ld_stream32(p, u[0], u[1]);
      } else {
        u[0] = ld_stream16(p);
        u[1] = ld_stream16(p + 8);
      }
    }
    at.next();
    constexpr uint32_t kAbs = 0x7FFF7FFFu;
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      m = max_nan_bf16x2(m, max_nan_bf16x2(max_nan_bf16x2(u[i].x & kAbs, u[i].y & kAbs),
                                           max_nan_bf16x2(u[i].z & kAbs, u[i].w & kAbs)));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m = max_nan_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t top = max(m & 0x7FFFu, (m >> 16) & 0x7FFFu);
    const bool finite = top < 0x7F80u;
    const float scale = finite ? over_127(fmaxf(__uint_as_float(top << 16), 1e-12f)) : __uint_as_float(0x7FC00000u);
    const F2 inv = f2(finite ? rcp_approx(scale) : 0.f);
    if (in) {
      uint32_t w[4] = {0u, 0u, 0u, 0u};
      if (finite) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t c[8];
          pack_pair(u[i].x, scale, inv, c[0], c[1]);
          pack_pair(u[i].y, scale, inv, c[2], c[3]);
          pack_pair(u[i].z, scale, inv, c[4], c[5]);
          pack_pair(u[i].w, scale, inv, c[6], c[7]);
#pragma unroll
          for (int q = 0; q < 2; ++q)
            w[2 * i + q] = prmt(prmt(c[4 * q], c[4 * q + 1], 0x0040u), prmt(c[4 * q + 2], c[4 * q + 3], 0x0040u), 0x5410u);
        }
      }
      *reinterpret_cast<uint4*>(codes + row * K + k) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (sub == 0 && row < M) scales[row * nrun + run] = scale;
  }
}

// Unpack: 16 codes per thread, two pieces in flight, 32 bytes per store where the
// rows are 32-byte aligned: 47 us at 6144 x 16384, 6.5 TB/s (8 codes and 16-byte
// stores: 51; four pieces of 16: 54; two of 8 on twice the resident CTAs: 59).
// The codes become bf16 exactly, so float32 by a shift, without integer
// conversions.
__device__ __forceinline__ uint4 restore8(uint32_t lo, uint32_t hi, F2 by) {
  uint4 p;
  i8_to_bf16(lo, p.x, p.y);
  i8_to_bf16(hi, p.z, p.w);
  return make_uint4(narrow(mul2(widen(p.x), by)), narrow(mul2(widen(p.y), by)), narrow(mul2(widen(p.z), by)),
                    narrow(mul2(widen(p.w), by)));
}
__global__ void __launch_bounds__(256)
    checkpoint_unpack_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                             int64_t M, int K, int nrun, bool wide, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  constexpr int kPieces = 2;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  RowWalk at(blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x, stride, K / 16);
  while (at.row < M) {
    uint4 u[kPieces];
    float s[kPieces];
    int64_t row[kPieces];
    int k[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      row[i] = at.row;
      k[i] = at.col * 16;
      if (row[i] < M) {
        u[i] = __ldg(reinterpret_cast<const uint4*>(codes + row[i] * K + k[i]));
        s[i] = __ldg(scales + row[i] * nrun + k[i] / kCkptRun);
      }
      at.next();
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (row[i] >= M) break;
      const F2 by = f2(s[i]);
      __nv_bfloat16* p = out + row[i] * ldo + k[i];
      const uint4 a = restore8(u[i].x, u[i].y, by), b = restore8(u[i].z, u[i].w, by);
      if (wide) {
        st_global32(p, a, b);
      } else {
        *reinterpret_cast<uint4*>(p) = a;
        *reinterpret_cast<uint4*>(p + 8) = b;
      }
    }
  }
}

}  // namespace dq
