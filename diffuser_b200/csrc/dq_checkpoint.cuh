// dq_checkpoint.cuh -- activations kept in 8 bits until the backward pass, and
// the transposed decode of a quantized weight for its input gradient
// (include/dq_adapter.h).
#pragma once

#include "dq_adapter.cuh"
#include "dq_codec.cuh"

namespace dq {

constexpr int kCkptRun = 128;  // features per scale

// Pack: 16 lanes per run of 128 features, 8 features (16 bytes) per lane, two
// runs per warp and two warps' worth of loads in flight.  The maximum is taken
// over the bit patterns of |x| (bf16 magnitudes order like integers, infinities
// and NaN above every number), so a run that is not finite is seen whatever the
// order.  HBM-bound: 3 bytes per feature; an IEEE division per feature made it
// 127 us at 6144 x 16384 (floor 47), so the quotient is taken as x (1 / scale),
// off by at most 127 (2^-24 + 2^-24) = 1.6e-5 from the exact one, and divided
// only where that could round to another integer: within 1e-4 of a half.
__device__ __forceinline__ uint32_t pack_code(float v, float scale, float inv) {
  const float t = v * inv;
  float q = rintf(t);
  if (fabsf(t - q) > 0.4999f) q = rintf(__fdiv_rn(v, scale));
  return static_cast<uint32_t>(static_cast<int>(q)) & 0xFFu;
}

__global__ void __launch_bounds__(256)
    checkpoint_pack_kernel(const __nv_bfloat16* __restrict__ x, int64_t ldx, int64_t runs, int nrun,
                           int K, int8_t* __restrict__ codes, float* __restrict__ scales) {
  const int half = (threadIdx.x & 31) >> 4, sub = threadIdx.x & 15;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 16;
  for (int64_t base = blockIdx.x * 16ll + (threadIdx.x >> 5) * 2; base < runs; base += 2 * stride) {
    uint4 u[2];
    int64_t row[2];
    int k[2];
    bool in[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t run = base + i * stride + half;
      row[i] = run / nrun;
      k[i] = static_cast<int>(run - row[i] * nrun) * kCkptRun + sub * 8;
      in[i] = run < runs && k[i] < K;
      u[i] = in[i] ? ld_stream16(x + row[i] * ldx + k[i]) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t m = __vmaxu2(__vmaxu2(u[i].x & 0x7FFF7FFFu, u[i].y & 0x7FFF7FFFu),
                            __vmaxu2(u[i].z & 0x7FFF7FFFu, u[i].w & 0x7FFF7FFFu));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint32_t top = max(m & 0xFFFFu, m >> 16);
      const bool finite = top < 0x7F80u;
      const float amax = fmaxf(__uint_as_float(top << 16), 1e-12f);
      const float scale = finite ? __fdiv_rn(amax, 127.0f) : __uint_as_float(0x7FC00000u);
      if (!in[i]) continue;
      uint32_t w[2] = {0u, 0u};
      if (finite) {
        const float inv = __frcp_rn(scale);
        float v[8];
        unpack8(u[i], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= pack_code(v[e], scale, inv) << (8 * (e & 3));
      }
      *reinterpret_cast<uint2*>(codes + row[i] * K + k[i]) = make_uint2(w[0], w[1]);
      if (sub == 0) scales[base + i * stride + half] = scale;
    }
  }
}

// Unpack: 8 codes per thread.
__global__ void __launch_bounds__(256)
    checkpoint_unpack_kernel(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                             int64_t M, int K, int nrun, __nv_bfloat16* __restrict__ out, int64_t ldo) {
  const int per_row = K / 8;
  const int64_t total = M * per_row;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x; i < total; i += stride) {
    const int64_t row = i / per_row;
    const int k = static_cast<int>(i - row * per_row) * 8;
    const uint2 u = *reinterpret_cast<const uint2*>(codes + row * K + k);
    const float s = __ldg(scales + row * nrun + k / kCkptRun);
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t w = e < 4 ? u.x : u.y;
      v[e] = static_cast<float>(static_cast<int8_t>(w >> (8 * (e & 3)))) * s;
    }
    *reinterpret_cast<uint4*>(out + row * ldo + k) = pack8(v);
  }
}

// ------------------------------------------------- transposed weight decode
// W [N, K] (NF4 or e4m3) -> bf16 W^T [K, N], the operand the bf16 pair GEMM
// takes for dx = dy . W.  A CTA decodes 128 weight rows x 64 k (one NF4 block
// per row): thread (pair p of rows, quarter kc of the 64 k) decodes 16 k of
// rows 2p and 2p + 1, pairs the two rows' values at each k with byte permutes
// and stores them at [k][p ^ 8 kc] (conflict-free: the four quarters of a row
// pair sit in distinct banks), then the CTA writes 256-byte row pieces of W^T.
// The values are those of dq_dequant_* bit for bit.
template <int FMT>
__global__ void __launch_bounds__(256)
    decode_transposed_kernel(const uint8_t* __restrict__ w, const void* __restrict__ absmax, int sbf,
                             float fp8_scale, int N, int K, __nv_bfloat16* __restrict__ out) {
  __shared__ __align__(16) uint32_t tile[64 * 64];  // [k][row pair]
  const int k0 = blockIdx.x * 64, n0 = blockIdx.y * 128;
  const int kc = threadIdx.x & 3, p = threadIdx.x >> 2;
  const int k = k0 + kc * 16;
  uint32_t o[2][8];  // 16 k of each row as bf16 pairs along k
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int n = n0 + 2 * p + h;
    if (n < N && k < K) {  // K is a multiple of 16
      if constexpr (FMT == kFmtNF4) {
        const uint2 u = *reinterpret_cast<const uint2*>(w + static_cast<int64_t>(n) * (K / 2) + k / 2);
        const Nf4Planes P =
            nf4_scaled_planes(nf4_scale2(load_scale(absmax, static_cast<int64_t>(n) * (K / 64) + k / 64, sbf != 0)));
        nf4_decode_word(u.x, P, o[h]);
        nf4_decode_word(u.y, P, o[h] + 4);
      } else {
        const float s = __bfloat162float(__float2bfloat16_rn(fp8_scale));
        const uint4 u = *reinterpret_cast<const uint4*>(w + static_cast<int64_t>(n) * K + k);
        fp8_decode_word(u.x, s, o[h]);
        fp8_decode_word(u.y, s, o[h] + 2);
        fp8_decode_word(u.z, s, o[h] + 4);
        fp8_decode_word(u.w, s, o[h] + 6);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[h][e] = 0u;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    tile[(kc * 16 + 2 * e) * 64 + (p ^ (8 * kc))] = prmt(o[0][e], o[1][e], 0x5410u);
    tile[(kc * 16 + 2 * e + 1) * 64 + (p ^ (8 * kc))] = prmt(o[0][e], o[1][e], 0x7632u);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (threadIdx.x >> 4) + 16 * i, ch = threadIdx.x & 15;  // 16-byte chunk of 8 weight rows
    const int n = n0 + ch * 8;
    if (k0 + row < K && n < N)  // N is a multiple of 8
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(k0 + row) * N + n) =
          *reinterpret_cast<const uint4*>(&tile[row * 64 + ((ch * 4) ^ (8 * (row >> 4)))]);
  }
}

}  // namespace dq
