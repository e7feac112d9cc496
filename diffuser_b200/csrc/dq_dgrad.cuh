// dq_dgrad.cuh -- input gradients of the quantized linears: dx = dy . W with W
// [N, K] kept as NF4 or e4m3 (include/dq_adapter.h).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cstdint>

#include "dq_codec.cuh"
#include "dq_f32x2.cuh"
#include "dq_internal.h"
#include "dq_tile.cuh"

namespace dq {

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

// ----------------------------------------------------------- decode and multiply
// For few tokens the two launches above cost more than the products: the
// decoded weight's way through memory, and a GEMM whose 256 x 256 tiles leave
// most SMs without one (333 x 4096 x 4096: 9.7 us and 20 us).  Here a CTA
// decodes a 128-feature slab of the weight into shared memory for up to 512
// tokens at once:
//
//   D[feature, token] += W[n, feature]^T dy[token, n], 64 n at a time.
//
// The weight's rows lie along the sum, so its decoded tile [64 n][128
// features] is the MMA's A operand with the features contiguous (MN-major, two
// blocks of 128-byte swizzled rows) and nothing is transposed; dy's boxes
// [tokens][64 n] come by TMA as the K-major B operand, the sums (f32) stay in
// tensor memory, up to all 512 columns.  Every weight element is decoded once.
// Eight warps decode (NF4 through the per-lane byte table: a lookup and a
// product per two weights), their weight words four steps ahead in registers,
// two issue the MMAs, one the TMA loads.
//
// The sum over N is split over the CTAs of a cluster so that the SMs have one
// CTA each; their partial sums meet through distributed shared memory, in rank
// order, and are rounded to bf16 once.
//
// Measured (NF4, against the two launches): 333 tokens x 4096 x 4096 20 us (28),
// one token 12.0 (26); 16384 x 4096: 46 (95), 31 (93).  A step of 64 n takes
// 0.40 us with few tokens, in which the decoding warps hardly wait, and 0.53 with
// 333, of the order of its shared-memory traffic (dy's boxes in and out, W's tile
// in and twice out, the table's lookups: some 150 KB).  Of the rest about 4 us
// are the sums' way out and 3 the first loads.
struct DgradArgs {
  const uint8_t* w;
  const void* absmax;
  __nv_bfloat16* dx;
  unsigned int* error;
  float fp8_scale;
  int scale_bf16;
  int M, N, K;
  int tok_n, n_mma;   // tokens per MMA (a multiple of 16, at most 256), MMAs per step (1 or 2)
  int stages, stage_bytes, per_split;
  int red_tokens;     // tokens whose f32 sums fit the ring
  uint32_t tmem_cols;
};

constexpr int kDgradRows = 64, kDgradFeatures = 128;
constexpr int kDgradWBytes = kDgradRows * kDgradFeatures * 2;
constexpr int kDgradMaxStages = 12;
constexpr int kDgradBars = 16 * kDgradMaxStages + 8;  // full, empty, done
constexpr int kDgradLutAt = 256;                      // the NF4 table, behind the barriers
constexpr int kDgradGroups = 2;                       // of four decoding warps
constexpr int kDgradMmaWarp = 4 * kDgradGroups, kDgradTmaWarp = kDgradMmaWarp + 2;  // two issue MMAs
constexpr int kDgradThreads = (kDgradTmaWarp + 1) * 32;

template <int FMT>
__global__ void __launch_bounds__(kDgradThreads, 1)
    dgrad_fused_kernel(const __grid_constant__ CUtensorMap tdy, const DgradArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw_base = smem_u32(smem_raw);
  const uint32_t sbase = (raw_base + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw_base);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int off_bar = a.stages * a.stage_bytes;
  auto full_bar = [&](int s) { return sbase + off_bar + 8u * s; };
  auto empty_bar = [&](int s) { return sbase + off_bar + 8u * (kDgradMaxStages + s); };
  const uint32_t done_bar = sbase + off_bar + 16u * kDgradMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + off_bar + kDgradBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + off_bar + kDgradBars + 8);
  if (tid == 0) {
    for (int s = 0; s < a.stages; ++s) {
      mbar_init(full_bar(s), 5);  // four decoding warps, the TMA issuer
      mbar_init(empty_bar(s), a.n_mma);
    }
    mbar_init(done_bar, a.n_mma);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if constexpr (FMT == kFmtNF4) nf4_lut_fill(reinterpret_cast<uint32_t*>(smem + off_bar + kDgradLutAt));
  if (warp == kDgradTmaWarp && lane == 0) prefetch_tensormap(&tdy);
  if (warp == kDgradMmaWarp) {
    tmem_alloc(smem_u32(tmem_slot), a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tokens = a.tok_n * a.n_mma;
  const int f0 = blockIdx.x * kDgradFeatures;
  const int me = blockIdx.y, ranks = gridDim.y;  // the cluster spans grid.y
  const int b_lo = me * a.per_split;
  const int steps = min((a.N + kDgradRows - 1) / kDgradRows, b_lo + a.per_split) - b_lo;  // at least one

  if (warp < kDgradMmaWarp) {
    // ---------------------------------------------------------------- decode
    // Two groups of four warps take the steps in turn, so that one's latencies
    // (barrier, lookups, the fence towards the MMAs) pass under the other's.
    // (No more groups than ring stages, of which there are at least two: a group
    // that comes to step i has seen step i - groups - stages consumed, and its
    // parity wait for i - stages is unambiguous only if i - 2 stages is among
    // those.  Four groups, where the ring has the stages: NF4 2-7% faster at
    // 12288 x 4096 and more, 3% slower at 4096 x 4096, e4m3 3% slower.)
    // This thread: 32 features (quarter q) of rows t / 4 and t / 4 + 32 of its
    // group's steps, the weight words two own steps ahead in registers.
    constexpr int kAhead = 2;
    const uint32_t lut_lane = sbase + a.stages * a.stage_bytes + kDgradLutAt + 4u * lane;
    constexpr int kWords = FMT == kFmtNF4 ? 1 : 2;
    const int group = warp >> 2, row0 = (tid & 127) >> 2, q = tid & 3;
    const int f = f0 + 32 * q;
    const bool swap = q >= 2;  // the second block's chunks in the order 2, 3, 0, 1: no bank twice
    const float s8 = FMT == kFmtFP8 ? __bfloat162float(__float2bfloat16_rn(a.fp8_scale)) : 0.f;
    struct Own {
      uint4 u[2][kWords];
      float scale[2];
    };
    // walking pointers: this thread's next row (and that + 32), of rows below
    // n_end (0: its features are past K; NF4's K % 64 == 0 puts a quarter all in
    // or all out, an e4m3 one's second half may be past it)
    const int64_t row_bytes = FMT == kFmtNF4 ? a.K / 2 : a.K;
    int n = (b_lo + group) * kDgradRows + row0;
    const int n_end = f < a.K ? min(a.N, (b_lo + steps) * kDgradRows) : 0;
    const bool upper = f + 16 < a.K;
    const uint8_t* src = a.w + n * row_bytes + (FMT == kFmtNF4 ? f / 2 : f);
    const int64_t src_step = static_cast<int64_t>(kDgradGroups) * kDgradRows * row_bytes;
    int64_t block = static_cast<int64_t>(n) * (a.K / 64) + f / 64;
    auto load = [&](Own& w) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool in = n + 32 * h < n_end;
        const uint4* p = reinterpret_cast<const uint4*>(src + 32 * h * row_bytes);
        w.u[h][0] = in ? __ldg(p) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (FMT == kFmtNF4)
          w.scale[h] = in ? load_scale(a.absmax, block + 32 * h * (a.K / 64), a.scale_bf16 != 0) : 0.f;
        else
          w.u[h][kWords - 1] = in && upper ? __ldg(p + 1) : make_uint4(0u, 0u, 0u, 0u);
      }
      n += kDgradGroups * kDgradRows;
      src += src_step;
      block += static_cast<int64_t>(kDgradGroups) * kDgradRows * (a.K / 64);
    };
    Own ahead[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) load(ahead[i]);
    int slot = group;
    uint32_t parity = 1;
    bool live = true;
    for (int base = group; base < steps && live; base += kDgradGroups * kAhead) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (base + kDgradGroups * i >= steps || !live) break;
        uint32_t o[2][16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (FMT == kFmtNF4) {
            // (rows past N have codes and a scale of zero: -1 times 0)
            const uint32_t sc2 = nf4_scale2(ahead[i].scale[h]);
            const uint4 u = ahead[i].u[h][0];
            nf4_decode_word_lut(swap ? u.z : u.x, lut_lane, sc2, o[h]);
            nf4_decode_word_lut(swap ? u.w : u.y, lut_lane, sc2, o[h] + 4);
            nf4_decode_word_lut(swap ? u.x : u.z, lut_lane, sc2, o[h] + 8);
            nf4_decode_word_lut(swap ? u.y : u.w, lut_lane, sc2, o[h] + 12);
          } else {
            const uint4 first = ahead[i].u[h][0], last = ahead[i].u[h][kWords - 1];
            const uint4 u = swap ? last : first, v = swap ? first : last;
            fp8_decode_word(u.x, s8, o[h]);
            fp8_decode_word(u.y, s8, o[h] + 2);
            fp8_decode_word(u.z, s8, o[h] + 4);
            fp8_decode_word(u.w, s8, o[h] + 6);
            fp8_decode_word(v.x, s8, o[h] + 8);
            fp8_decode_word(v.y, s8, o[h] + 10);
            fp8_decode_word(v.z, s8, o[h] + 12);
            fp8_decode_word(v.w, s8, o[h] + 14);
          }
        }
        load(ahead[i]);
        if (!mbar_wait(empty_bar(slot), parity, abort_flag)) {
          live = false;
          break;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int row = row0 + 32 * h;
          const uint32_t at = sbase + slot * a.stage_bytes + (q >> 1) * (kDgradWBytes / 2) + row * 128;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int chunk = 4 * (q & 1) + (swap ? j ^ 2 : j);
            sts128(at + ((chunk ^ (row & 7)) << 4),
                   make_uint4(o[h][4 * j], o[h][4 * j + 1], o[h][4 * j + 2], o[h][4 * j + 3]));
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(slot));
        slot += kDgradGroups;
        if (slot >= a.stages) {
          slot -= a.stages;
          parity ^= 1u;
        }
      }
    }
  } else if (warp < kDgradTmaWarp) {
    // ------------------------------------------------------------------- MMA
    // Each half of more than 256 tokens, with its own sums, has its own issuing
    // thread (one for both: 333 x 4096 x 4096 20.4 us, two 20.0; two halves for
    // fewer tokens read W's tile twice: 16384 x 4096 3% slower)
    const int m = warp - kDgradMmaWarp;
    if (m < a.n_mma && lane == 0) {
      const uint32_t idesc = make_idesc_bf16(128, a.tok_n) | (1u << 15);  // A MN-major
      const uint32_t d = tmem + m * a.tok_n, x_at = kDgradWBytes + m * a.tok_n * 128;
      uint32_t at = sbase, parity = 0;
      int slot = 0;
      for (int it = 0; it < steps; ++it) {
        if (!mbar_wait(full_bar(slot), parity, abort_flag)) break;
        tc_fence_after();
        const uint64_t ad = make_sw128_mnmajor_desc(at, kDgradWBytes / 2);
        const uint64_t bd = make_sw128_kmajor_desc(at + x_at);
#pragma unroll
        for (int ks = 0; ks < 4; ++ks)  // 16 n: two 8-row groups of W, 32 bytes of dy's rows
          tc_mma_ss(d, ad + 128 * ks, bd + 2 * ks, idesc, (it | ks) != 0);
        tc_commit(empty_bar(slot));
        at += a.stage_bytes;
        if (++slot == a.stages) {
          slot = 0;
          at = sbase;
          parity ^= 1u;
        }
      }
      tc_commit(done_bar);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------------- TMA
    if (lane == 0) {
      uint32_t dst = sbase + kDgradWBytes, parity = 1;
      int slot = 0;
      for (int it = 0; it < steps; ++it) {
        if (!mbar_wait(empty_bar(slot), parity, abort_flag)) break;
        mbar_arrive_expect_tx(full_bar(slot), static_cast<uint32_t>(tokens * 128));
        for (int m = 0; m < a.n_mma; ++m)
          tma_load_2d(dst + m * a.tok_n * 128, &tdy, full_bar(slot), (b_lo + it) * kDgradRows, m * a.tok_n);
        dst += a.stage_bytes;
        if (++slot == a.stages) {
          slot = 0;
          dst = sbase + kDgradWBytes;
          parity ^= 1u;
        }
      }
    }
    __syncwarp();
  }
  // partial sums [tokens][128 features] f32 in this CTA's (drained) ring
  float* red = reinterpret_cast<float*>(smem);
  const bool ok = mbar_wait(done_bar, 0, abort_flag);
  tc_fence_after();
  __syncthreads();
  for (int t0 = 0; t0 < tokens; t0 += a.red_tokens) {
    const int tn = min(a.red_tokens, tokens - t0);
    if (ok && warp < kDgradMmaWarp) {
      const int quad = warp & 3;
      for (int c = (warp >> 2) * 16; c < tn; c += 16 * kDgradGroups) {
        uint32_t v[16];
        tmem_ld_x16(tmem + (static_cast<uint32_t>(32 * quad) << 16) + t0 + c, v);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 16; ++e) red[(c + e) * kDgradFeatures + 32 * quad + lane] = __uint_as_float(v[e]);
      }
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync();
    const int per = (tn + ranks - 1) / ranks;
    const int hi = min(min(tn, (me + 1) * per), a.M - t0);
    const int f = f0 + 4 * lane;
    if (!*abort_flag && f < a.K) {
      // eight loads at a time: 8 / ranks rows (ranks is a power of two) of every rank
      constexpr int kWarps = kDgradThreads / 32;
      const int shift = 31 - __clz(ranks), rows = 8 >> shift;
      for (int i = me * per + warp; i < hi; i += rows * kWarps) {
        float4 u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = i + (e >> shift) * kWarps;
          if (row < hi)
            u[e] = ld_cluster_f4(mapa_shared(sbase + static_cast<uint32_t>(row * kDgradFeatures + 4 * lane) * 4u,
                                             e & (ranks - 1)));
        }
        F2 lo = f2(0.f), up = f2(0.f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int row = i + (e >> shift) * kWarps;
          if ((e & (ranks - 1)) == 0) lo = up = f2(0.f);
          lo = add2(lo, f2(u[e].x, u[e].y));
          up = add2(up, f2(u[e].z, u[e].w));
          if ((e & (ranks - 1)) == ranks - 1 && row < hi)
            *reinterpret_cast<uint2*>(a.dx + static_cast<int64_t>(t0 + row) * a.K + f) =
                make_uint2(narrow(lo), narrow(up));
        }
      }
    }
    __syncwarp();
    cluster_sync();  // every rank has read this one's sums
  }
  if (*abort_flag) {  // let loads in flight land before this CTA's memory goes
    const unsigned long long t0 = globaltimer_ns();
    while (globaltimer_ns() - t0 < 200000ull) {
    }
    if (tid == 0) atomicOr(a.error, 1u << kErrTimeout);
  }
  __syncthreads();
  if (warp == kDgradMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, a.tmem_cols);
  }
}

}  // namespace dq
