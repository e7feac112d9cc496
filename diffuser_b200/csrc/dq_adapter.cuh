// dq_adapter.cuh -- low-rank adapters beside the quantized linears
// (include/dq_adapter.h).
//
// Mathematics.  With the adapters' factors both stored [r, features], every
// product of the forward and the backward pass is one of three:
//   down   v[m, :] = X[m, :] . P_a^T          (x with down; dy with up)
//   up     O[m, :] = Y[m, :] + s_a v[m, :] . P_a   (y with up; dx with down)
//   wgrad  dP_a    = sum_m G[m, :]^T X[m, :]  (hidden with dy; g with x)
// where a is the adapter of token m.  r <= 128 against thousands of features,
// so all three are bound by the one wide operand's bytes (X; Y read and O
// written), not by the multiplications: 2 r FLOP per 2-byte element of X is
// 64 FLOP/B at r = 64, against the machine's 256.  Everything is arranged around
// the stream of the wide operand: each element of it is read once per kernel, in
// 16-byte pieces, several stages ahead.  down and wgrad, which at r = 64 ask for
// more than the warp-level MMAs give (about 320 TFLOP/s measured), sum in tensor
// memory; up, whose sums meet Y element by element, in registers.
//
// Plan.  Tokens are visited sorted by adapter, each adapter's run padded to a
// multiple of 16 rows with -1 entries, so that every 16-row MMA block belongs
// to one adapter and no product ever mixes rows of two; padded rows are
// loaded as zeros (never multiplied by zero: a NaN in a neighbour's row does
// not travel).  The last bucket holds the tokens without an adapter.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "dq_codec.cuh"
#include "dq_f32x2.cuh"
#include "dq_internal.h"
#include "dq_ptx.cuh"
#include "dq_smallm.cuh"
#include "dq_tile.cuh"

namespace dq {

// ------------------------------------------------------------------ the plan
constexpr int kTileRows = 128;  // rows of a large tile
constexpr int kBlockRows = 16;  // rows of an MMA block, and of a small tile

// int32 words of the plan buffer
struct AdapterPlan {
  // header words
  static constexpr int kRows = 0;       // rows in use (16-row multiples, all buckets)
  static constexpr int kNoneStart = 1;  // first row of the tokens without an adapter
  static constexpr int kTiles = 2;      // large tiles with an adapter
  static constexpr int kAllTiles = 3;   // large tiles of all buckets
  static constexpr int kHeader = 16;
  int64_t cap, max_tiles;
  int64_t off_start, off_counts, off_perm, off_blk, off_tiles, words;
};

// Buckets that can hold tokens: at most min(A, R) adapters and the rest.
__host__ __device__ inline AdapterPlan adapter_plan_layout(int64_t M, int64_t R, int A) {
  AdapterPlan p;
  const int64_t groups = (A < R ? A : R) + 1;
  p.cap = (M + 15 * groups + 15) / 16 * 16;
  p.max_tiles = p.cap / kTileRows + groups;
  auto up4 = [](int64_t v) { return (v + 3) / 4 * 4; };
  p.off_start = AdapterPlan::kHeader;
  p.off_counts = p.off_start + up4(A + 2);
  p.off_perm = p.off_counts + up4(A + 1);
  p.off_blk = p.off_perm + p.cap;  // cap is a multiple of 16
  p.off_tiles = p.off_blk + up4(p.cap / 16);
  p.words = p.off_tiles + 4 * p.max_tiles;
  return p;
}

// Requests seen as R + 2 runs: the tokens before the first, the requests, the
// tokens behind the last.  Bucket of a run: its adapter, or A for none.
struct RunList {
  const int32_t* ids;
  const int32_t* offsets;
  int R, M, A;
  bool valid;  // offsets are in order and within 0..M
  __device__ __forceinline__ void run(int j, int* bucket, int* start, int* len) const {
    *bucket = A;
    if (!valid) {  // every token in one run without an adapter
      *start = 0;
      *len = j == 0 ? M : 0;
      return;
    }
    const int lo = j == 0 ? 0 : offsets[j - 1];
    const int hi = j == R + 1 ? M : offsets[j];
    *start = lo;
    *len = hi - lo;
    if (j >= 1 && j <= R) {
      const int id = ids[j - 1];
      if (id >= 0 && id < A) *bucket = id;
    }
  }
};

// Whether the offsets are in order (every thread of the CTA gets the answer);
// CTA 0 records what is out of range.
__device__ __forceinline__ bool check_runs(const RunList& q, unsigned int* error) {
  int bad = 0, bad_id = 0;
  for (int j = threadIdx.x; j <= q.R; j += blockDim.x) {
    const int o = q.offsets[j];
    if (o < 0 || o > q.M || (j > 0 && o < q.offsets[j - 1])) bad = 1;
    if (j < q.R && (q.ids[j] < -1 || q.ids[j] >= q.A)) bad_id = 1;
  }
  bad = __syncthreads_or(bad);
  bad_id = __syncthreads_or(bad_id);
  if ((bad || bad_id) && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(error, 1u << kErrIndex);
  return bad == 0;
}

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Rows of each bucket: one warp per bucket walks all runs.
__global__ void __launch_bounds__(256)
    adapter_count_kernel(const int32_t* __restrict__ ids, const int32_t* __restrict__ offsets, int R,
                         int M, int A, int32_t* __restrict__ counts, unsigned int* error) {
  RunList q{ids, offsets, R, M, A, true};
  q.valid = check_runs(q, error);
  const int lane = threadIdx.x & 31;
  const int a = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (a > A) return;
  int n = 0;
  for (int j = lane; j < R + 2; j += 32) {
    int b, start, len;
    q.run(j, &b, &start, &len);
    if (b == a) n += len;
  }
  n = warp_sum(n);
  if (lane == 0) counts[a] = n;
}

// Places each bucket's tokens, in order, behind the buckets before it.
__global__ void __launch_bounds__(256)
    adapter_place_kernel(const int32_t* __restrict__ ids, const int32_t* __restrict__ offsets, int R,
                         int M, int A, int32_t* __restrict__ words, AdapterPlan lay, unsigned int* error) {
  RunList q{ids, offsets, R, M, A, true};
  q.valid = check_runs(q, error);
  const int lane = threadIdx.x & 31;
  const int a = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  if (a > A) return;
  const int32_t* counts = words + lay.off_counts;
  int row0 = 0, tile0 = 0;
  for (int b = lane; b < a; b += 32) {
    const int c = counts[b];
    row0 += (c + 15) / 16 * 16;
    tile0 += (c + kTileRows - 1) / kTileRows;
  }
  row0 = warp_sum(row0);
  tile0 = warp_sum(tile0);
  const int mine = counts[a], rows = (mine + 15) / 16 * 16;
  int32_t* perm = words + lay.off_perm;
  int at = row0;
  for (int base = 0; base < R + 2; base += 32) {
    const int j = base + lane;
    int b = -1, start = 0, len = 0;
    if (j < R + 2) q.run(j, &b, &start, &len);
    if (b != a) len = 0;
    int before = len;  // inclusive scan of the lengths
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    const int total = __shfl_sync(0xffffffffu, before, 31);
    before -= len;
    // short runs by their own lane, long ones by the whole warp
    for (int i = 0; i < len && i < 4; ++i) perm[at + before + i] = start + i;
    unsigned int rest = __ballot_sync(0xffffffffu, len > 4);
    while (rest != 0) {
      const int src = __ffs(rest) - 1;
      rest &= rest - 1;
      const int s = __shfl_sync(0xffffffffu, start, src);
      const int l = __shfl_sync(0xffffffffu, len, src);
      const int p = __shfl_sync(0xffffffffu, before, src);
      for (int i = 4 + lane; i < l; i += 32) perm[at + p + i] = s + i;
    }
    at += total;
  }
  for (int i = mine + lane; i < rows; i += 32) perm[row0 + i] = -1;
  for (int i = lane; i < rows / 16; i += 32) words[lay.off_blk + row0 / 16 + i] = a;
  const int tiles = (mine + kTileRows - 1) / kTileRows;
  // large tiles: first row, rows with a token, bucket, and the first token if
  // the tile's tokens follow one another (their readers then skip perm), else -1
  __syncwarp();
  for (int i = 0; i < tiles; ++i) {
    const int r0 = row0 + i * kTileRows, n = min(kTileRows, mine - i * kTileRows);
    const int first = perm[r0];
    bool run = true;
    for (int j = lane; j < n; j += 32) run = run && perm[r0 + j] == first + j;
    run = __all_sync(0xffffffffu, run);
    if (lane == 0) reinterpret_cast<int4*>(words + lay.off_tiles)[tile0 + i] = make_int4(r0, n, a, run ? first : -1);
  }
  if (lane == 0) {
    words[lay.off_start + a] = row0;
    if (a == A) {
      words[lay.off_start + A + 1] = row0 + rows;
      words[AdapterPlan::kRows] = row0 + rows;
      words[AdapterPlan::kNoneStart] = row0;
      words[AdapterPlan::kTiles] = tile0;
      words[AdapterPlan::kAllTiles] = tile0 + tiles;
    }
  }
}

// One tile of up to T rows of one bucket; rows == 0: none for this CTA.
struct PlanTile {
  int row, rows, adapter;
  int first;  // large tiles: the first token if they follow one another, else -1
  // token of row i, or -1
  __device__ __forceinline__ int token(const int32_t* perm, int i) const {
    return i >= rows ? -1 : first >= 0 ? first + i : perm[row + i];
  }
};
template <int T>
__device__ __forceinline__ PlanTile plan_tile(const int32_t* words, const AdapterPlan& lay, int A,
                                              int tile, bool with_none) {
  PlanTile t{0, 0, A, -1};
  if constexpr (T == kTileRows) {
    const int count = words[with_none ? AdapterPlan::kAllTiles : AdapterPlan::kTiles];
    const int4 e = __ldg(reinterpret_cast<const int4*>(words + lay.off_tiles) + tile);  // grid <= max_tiles
    if (tile >= count) return t;
    t.row = e.x;
    t.rows = e.y;
    t.adapter = e.z;
    t.first = e.w;
  } else {
    t.row = tile * T;
    const int count = words[with_none ? AdapterPlan::kRows : AdapterPlan::kNoneStart];
    const int adapter = words[lay.off_blk + tile];  // grid <= cap / 16
    if (t.row >= count) return t;
    t.adapter = adapter;
    t.rows = T;
  }
  return t;
}

// ------------------------------------------------------------------- down
// hidden[token, :] = bf16(s_a X[token, :] . P_a^T), and f32 unrounded for the
// caller that multiplies it further.
//
// Large tiles: 128 rows, D = X P^T on tcgen05 (M = 128, N = R, f32 in tensor
// memory).  The stream of X needs 2 r FLOP per 2 bytes, 412 TFLOP/s at r = 64
// and the copy bandwidth; warp-level MMAs stop at about 320 here (measured:
// r = 64, 4608 x 12288, 55 us, 2.0 TB/s, with their pipe 41% busy and the
// rest of the time in fragment loads), the tensor-memory ones are free next
// to the stream.  Eight warps copy 64-feature stages with cp.async (the rows
// are gathered through the plan; 128-byte rows, 16-byte chunk c of row i at
// c ^ (i % 8), the 128-byte swizzle the MMA descriptors name), each thread
// several stages ahead: its copies of a stage are waited for, fenced towards
// the async proxy and reported to the stage's barrier when it issues the one
// kAhead later (two less than the ring, so that the MMAs of the stage to be
// refilled are not waited for).  A ninth warp issues the MMAs.
//
// The features are split over the CTAs of a cluster (enough of them to give
// every SM a CTA); their partial sums meet through distributed shared memory,
// in rank order, so nothing but the bf16 result reaches global memory.
//
// Measured: 4608 x 12288 at r = 64 31 us, of which the loop takes 25 (X at 4.5
// TB/s, and P, a third of every stage, from L2) and the cluster's sums 6; 4613
// x 4096 at r = 32 12 us.  TMA boxes for tiles of consecutive tokens, prefetches
// to L2 ten stages ahead, ranks that take 64-feature blocks in turn and 200 KB
// rings (whose clusters then run in two waves) were each within 3% or slower.
template <int R>
struct DownCfg {
  static constexpr int kStageX = kTileRows * 128;
  static constexpr int kStage = kStageX + R * 128;
  static constexpr int kStages = 110 * 1024 / kStage;  // two CTAs per SM
  static constexpr int kAhead = kStages - 2;           // stages a thread's copies run ahead
  static constexpr int kProducers = 8;
  static constexpr int kThreads = (kProducers + 1) * 32;
  static constexpr int kRedStride = R + 4;  // floats; conflict-free 16-byte rows
  static constexpr int kOffBar = kStages * kStage;
  static constexpr int kSmemBytes = kOffBar + 16 * kStages + 32 + 1024;
  static constexpr int kTmemCols = R < 32 ? 32 : R;
  static_assert(kTileRows * kRedStride * 4 <= kStages * kStage, "the sums fit the drained ring");
};

struct DownArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* bank;
  const float* scale;
  const int32_t* words;
  __nv_bfloat16* hidden;  // [M, rank]
  float* hidden32;        // [M, rank] or NULL
  unsigned int* error;
  AdapterPlan lay;
  int64_t ldx;
  int K, rank, A, k_per_split;
};

template <int R>
__global__ void __launch_bounds__(DownCfg<R>::kThreads, 2) adapter_down_kernel(const DownArgs a) {
  using C = DownCfg<R>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  const PlanTile t = plan_tile<kTileRows>(a.words, a.lay, a.A, blockIdx.x, false);
  if (t.rows == 0) return;  // the whole cluster: it shares the tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto full_bar = [&](int s) { return sbase + C::kOffBar + 8u * s; };
  auto empty_bar = [&](int s) { return sbase + C::kOffBar + 8u * (C::kStages + s); };
  const uint32_t done_bar = sbase + C::kOffBar + 16u * C::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffBar + 16 * C::kStages + 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffBar + 16 * C::kStages + 16);
  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full_bar(s), C::kProducers);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == C::kProducers) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_launch_dependents();
  const int k_lo = blockIdx.y * a.k_per_split;
  const int k_hi = min(a.K, k_lo + a.k_per_split);
  const int steps = (k_hi - k_lo + 63) / 64;

  if (warp < C::kProducers) {
    const __nv_bfloat16* P = a.bank + static_cast<int64_t>(t.adapter) * a.rank * a.K;
    const int chunk = tid & 7;  // this thread copies chunk tid % 8 of rows tid / 8 + 32 i
    const __nv_bfloat16* src[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (tid >> 3) + 32 * i;
      const int token = t.token(a.words + a.lay.off_perm, row);
      src[i] = token >= 0 ? a.x + static_cast<int64_t>(token) * a.ldx : nullptr;
    }
    int it = 0;
    for (; it < steps; ++it) {
      const int slot = it % C::kStages;
      if (!mbar_wait(empty_bar(slot), static_cast<uint32_t>(((it / C::kStages) & 1) ^ 1), abort_flag)) break;
      const uint32_t sx = sbase + slot * C::kStage, sp = sx + C::kStageX;
      const int k = k_lo + it * 64 + chunk * 8;
      const bool in = k < k_hi;
      // rows without a token keep whatever the stage holds: row i of X only
      // reaches row i of D, which is not stored then
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = (tid >> 3) + 32 * i;
        if (src[i] != nullptr) cp_async_16_l2(sx + row * 128 + ((chunk ^ (row & 7)) << 4), in ? src[i] + k : a.x, in);
      }
#pragma unroll
      for (int i = 0; i < (R * 8 + 255) / 256; ++i) {
        const int row = (tid >> 3) + 32 * i;
        const bool ok = in && row < a.rank;
        if (row < R)
          cp_async_16(sp + row * 128 + ((chunk ^ (row & 7)) << 4),
                      ok ? P + static_cast<int64_t>(row) * a.K + k : a.bank, ok);
      }
      cp_async_commit();
      if (it >= C::kAhead) {
        cp_async_wait<C::kAhead>();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar((it - C::kAhead) % C::kStages));
      }
    }
    cp_async_wait<0>();
    fence_proxy_async_smem();
    __syncwarp();
    if (it == steps && lane == 0)
      for (int s = max(0, steps - C::kAhead); s < steps; ++s) mbar_arrive(full_bar(s % C::kStages));
  } else {
    constexpr uint32_t idesc = make_idesc_bf16(128, R);
    int it = 0;
    for (; it < steps; ++it) {
      const int slot = it % C::kStages;
      if (!mbar_wait(full_bar(slot), static_cast<uint32_t>((it / C::kStages) & 1), abort_flag)) break;
      tc_fence_after();
      const uint64_t ad = make_sw128_kmajor_desc(sbase + slot * C::kStage);
      const uint64_t bd = make_sw128_kmajor_desc(sbase + slot * C::kStage + C::kStageX);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) tc_mma_ss_elect(tmem, ad + 2 * ks, bd + 2 * ks, idesc, (it | ks) != 0);
      tc_commit_elect(empty_bar(slot));
    }
    tc_commit_elect(done_bar);
    __syncwarp();
  }
  // partial sums [128][R] f32 in this CTA's (drained) ring
  float* red = reinterpret_cast<float*>(smem);
  const bool ok = mbar_wait(done_bar, 0, abort_flag);
  tc_fence_after();
  constexpr int kHalves = R >= 32 ? 2 : 1;
  constexpr int kCols = R / kHalves;
  if (ok && warp < 4 * kHalves) {
    const int q = warp & 3, c0 = (warp >> 2) * kCols;
    float* dst = red + (32 * q + lane) * C::kRedStride + c0;
#pragma unroll
    for (int c = 0; c < kCols; c += 16) {
      uint32_t v[16];
      tmem_ld_x16(tmem + (static_cast<uint32_t>(32 * q) << 16) + c0 + c, v);
      tmem_wait_ld();
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<uint4*>(dst + c + e) = make_uint4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();
  const int ranks = gridDim.y, me = blockIdx.y;  // the cluster spans grid.y
  const int per = (t.rows + ranks - 1) / ranks;
  const int row_hi = min(t.rows, (me + 1) * per);
  const float s = a.scale[t.adapter];
  if (!*abort_flag) {
    for (int i = me * per * (R / 4) + tid; i < row_hi * (R / 4); i += C::kThreads) {
      const int row = i / (R / 4), c = (i % (R / 4)) * 4;
      const int token = t.token(a.words + a.lay.off_perm, row);
      if (c >= a.rank) continue;
      const uint32_t at = sbase + static_cast<uint32_t>(row * C::kRedStride + c) * 4u;
      float4 u[8];  // every rank's loads before the first sum
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < ranks) u[q] = ld_cluster_f4(mapa_shared(at, q));
      float v[4] = {};
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (q < ranks) {
          v[0] += u[q].x;
          v[1] += u[q].y;
          v[2] += u[q].z;
          v[3] += u[q].w;
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] *= s;
      const int64_t o = static_cast<int64_t>(token) * a.rank + c;
      *reinterpret_cast<uint2*>(a.hidden + o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      if (a.hidden32 != nullptr) *reinterpret_cast<float4*>(a.hidden32 + o) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  __syncwarp();
  cluster_sync();  // the other ranks have read this one's sums
  if (tid == 0 && *abort_flag) atomicOr(a.error, 1u << kErrTimeout);
  if (warp == C::kProducers) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Activations of the sum y + delta, float32 in and out (rounded once, with the
// result): gelu_tanh(x) = x sigmoid(2 u), u = sqrt(2/pi) (x + 0.044715 x^3), and
// silu(x) = x sigmoid(x), sigmoid(z) = 1 / (1 + 2^(-z log2 e)): an exponential
// and a reciprocal of the special-function unit, whose 16 results a cycle and
// SM stay below the stream's time (2^inf gives 1 / inf = 0: no clamp).
// Two at a time, the products in packed instructions.
__device__ __forceinline__ F2 sigmoid2_of_neg_log2(F2 z) {
  const float2 e = unpair(z);
  const float2 d = unpair(add2(f2(exp2f_approx(e.x), exp2f_approx(e.y)), f2(1.0f)));
  return f2(rcp_approx(d.x), rcp_approx(d.y));
}
__device__ __forceinline__ F2 gelu_tanh2(F2 x) {
  constexpr float k = -2.0f * 0.7978845608028654f * 1.4426950408889634f;
  return mul2(x, sigmoid2_of_neg_log2(mul2(x, fma2(mul2(x, x), f2(0.044715f * k), f2(k)))));
}
__device__ __forceinline__ F2 silu2(F2 x) { return mul2(x, sigmoid2_of_neg_log2(mul2(x, f2(-1.4426950408889634f)))); }
__device__ __forceinline__ F2 gate2(F2 x, int act) { return act == kActSwiGlu ? silu2(x) : gelu_tanh2(x); }

// --------------------------------------------------------------------- up
// O[m, :] = act(Y[m, :] + hidden[m, :] . P_a): 128-row tiles, one warp per 16.
//
// Bound: the stream of Y and O (P and hidden are small and reread from L2).
// The products take a sixteenth of the warp MMA rate at the copy bandwidth,
// so they stay warp-level with their sums in registers, and what counts is
// that nothing waits and that few instructions surround the stream: Y and P
// arrive by cp.async in a ring of 64-column steps, two ahead; Y's tile is read
// as accumulators with ldmatrix (its fragment is the MMA's own layout), the
// result returns to the same place with stmatrix and leaves in whole 128-byte
// rows.  A warp touches only its own 16 rows of Y and O, so the one barrier
// of a step is the ring's.
//
// Measured: 4613 x 16384 at r = 32 with GELU, down product included, 77 us (302
// MB of Y and O; a copy in the same pieces takes 53), 67 without.  No unit is the
// bound: issue slots 56% busy, the special-function unit 58 (two results per
// element), shared memory 53, DRAM 45; the stalls are fixed latencies and the
// shared-memory pipe at 24 warps per SM.  (Products onto zeros and Y added
// behind them in another thread layout, P scattered into place by 4-byte stores:
// 80 and 74.  One wave of CTAs with equal shares of all column steps: 78.)
template <int R>
struct UpCfg {
  static constexpr int kStepCols = 64;
  static constexpr int kYStage = kTileRows * kStepCols * 2;
  static constexpr int kStage = kYStage + R * kStepCols * 2;
  static constexpr int kStages = 3;
  static constexpr int kSmemBytes = kStages * kStage;
  static constexpr int kMinCtas = R <= 16 ? 4 : R <= 64 ? 3 : 2;
};

struct UpArgs {
  const __nv_bfloat16* y;
  const __nv_bfloat16* bank;
  const __nv_bfloat16* hidden;
  const int32_t* words;
  __nv_bfloat16* out;
  __nv_bfloat16* zero_hidden;  // rows without an adapter are zeroed here (or NULL)
  AdapterPlan lay;
  int64_t ldy, ldo;
  int N, rank, A, act, with_none, cols_per_cta;
};

template <int R>
__global__ void __launch_bounds__(256, UpCfg<R>::kMinCtas) adapter_up_kernel(const UpArgs a) {
  using C = UpCfg<R>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const PlanTile t = plan_tile<kTileRows>(a.words, a.lay, a.A, blockIdx.x, a.with_none != 0);
  if (t.rows == 0) {
    grid_wait();  // no CTA ends before the grid it depends on
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, tig = lane & 3;
  const int n_lo = blockIdx.y * a.cols_per_cta;
  const int n_hi = min(a.N, n_lo + a.cols_per_cta);
  const bool none = t.adapter >= a.A, gated = act_is_gated(a.act);
  const int32_t* perm = a.words + a.lay.off_perm;
  const __nv_bfloat16* P = a.bank + static_cast<int64_t>(none ? 0 : t.adapter) * a.rank * a.N;
  // this lane moves chunk lane % 8 of its warp's rows lane / 8 + 4 i (gated
  // results: chunk lane % 4 of rows lane / 4 + 8 i)
  const int ch = lane & 7;
  const __nv_bfloat16* ysrc[4];
  __nv_bfloat16* dst[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tok = t.token(perm, warp * 16 + (lane >> 3) + 4 * i);
    ysrc[i] = tok >= 0 ? a.y + static_cast<int64_t>(tok) * a.ldy + ch * 8 : nullptr;
    const int to = !gated ? tok : i < 2 ? t.token(perm, warp * 16 + g4 + 8 * i) : -1;
    dst[i] = to >= 0 ? a.out + static_cast<int64_t>(to) * a.ldo + (gated ? tig : ch) * 8 : nullptr;
  }
  auto load = [&](int n0, int stage) {
    const bool in = n0 + ch * 8 < n_hi;
    const uint32_t sy = sbase + stage * C::kStage, sp = sy + C::kYStage;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = warp * 16 + (lane >> 3) + 4 * i;
      if (in && ysrc[i] != nullptr) cp_async_16_l2(sy + row * 128 + ((ch ^ (row & 7)) << 4), ysrc[i] + n0, true);
    }
    if (!none && n0 < n_hi) {
#pragma unroll
      for (int i = 0; i < (R * 8 + 255) / 256; ++i) {
        const int row = (tid >> 3) + 32 * i;
        const bool ok = in && row < a.rank;
        if (R % 32 == 0 || row < R)
          cp_async_16(sp + row * 128 + ((ch ^ (row & 7)) << 4),
                      ok ? P + static_cast<int64_t>(row) * a.N + n0 + ch * 8 : a.bank, ok);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kStages - 1; ++i) load(n_lo + i * C::kStepCols, i);

  grid_wait();  // hidden is the down kernel's
  uint32_t vf[R / 16][4];
  {
    const int tok0 = t.token(perm, warp * 16 + g4), tok1 = t.token(perm, warp * 16 + g4 + 8);
#pragma unroll
    for (int ks = 0; ks < R / 16; ++ks)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = ks * 16 + 8 * (q >> 1);
        const int tok = (q & 1) ? tok1 : tok0;
        const bool ok = tok >= 0 && c < a.rank;
        const int64_t o = static_cast<int64_t>(tok) * a.rank + c + 2 * tig;
        vf[ks][q] = ok && !none ? __ldcg(reinterpret_cast<const unsigned int*>(a.hidden + o)) : 0u;
        if (ok && none && a.zero_hidden != nullptr && blockIdx.y == 0)
          *reinterpret_cast<uint32_t*>(a.zero_hidden + o) = 0u;
      }
  }
  grid_launch_dependents();

  // ldmatrix / stmatrix address of this lane: row lane % 16 of 16, column half lane / 16
  const int lrow = lane & 15, lhalf = lane >> 4;
  int stage = 0;
  for (int n0 = n_lo; n0 < n_hi; n0 += C::kStepCols) {
    cp_async_wait<C::kStages - 2>();
    __syncthreads();  // this step's Y and P; every warp is done with the last step's
    load(n0 + (C::kStages - 1) * C::kStepCols, stage == 0 ? C::kStages - 1 : stage - 1);
    const uint32_t sy = sbase + stage * C::kStage, sp = sy + C::kYStage;
    const uint32_t ybase = sy + (warp * 16 + lrow) * 128;
    auto at = [&](int chunk) { return ybase + (((chunk + lhalf) ^ (lrow & 7)) << 4); };
#pragma unroll
    for (int g = 0; g < 2; ++g) {  // 32 columns: four n-tiles of 8, their sums started from Y (widened exactly)
      float acc[4][4];
#pragma unroll
      for (int jp = 0; jp < 2; ++jp) {
        uint32_t w[4];
        ldmatrix_x4(at(4 * g + 2 * jp), w);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          acc[2 * jp + (q >> 1)][2 * (q & 1)] = __uint_as_float(w[q] << 16);
          acc[2 * jp + (q >> 1)][2 * (q & 1) + 1] = __uint_as_float(w[q] & 0xFFFF0000u);
        }
      }
      if (!none) {
#pragma unroll
        for (int ks = 0; ks < R / 16; ++ks)
#pragma unroll
          for (int jp = 0; jp < 2; ++jp) {
            uint32_t bf[4];
            ldmatrix_x4_trans(sp + (ks * 16 + lrow) * 128 + (((4 * g + 2 * jp + lhalf) ^ (lrow & 7)) << 4), bf);
            mma_16816_bf16(acc[2 * jp], vf[ks][0], vf[ks][1], vf[ks][2], vf[ks][3], bf[0], bf[1]);
            mma_16816_bf16(acc[2 * jp + 1], vf[ks][0], vf[ks][1], vf[ks][2], vf[ks][3], bf[2], bf[3]);
          }
      }
      F2 v[4][2];  // [n-tile][row half]
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) v[j][h] = f2(acc[j][2 * h], acc[j][2 * h + 1]);
      if (gated) {  // n-tiles 0, 1 hold 16 gate columns, 2, 3 their up columns
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int h = 0; h < 2; ++h) v[j][h] = mul2(gate2(v[j][h], a.act), v[j + 2][h]);
        stmatrix_x4(at(2 * g), narrow(v[0][0]), narrow(v[0][1]), narrow(v[1][0]), narrow(v[1][1]));
      } else {
        if (a.act == kActGeluTanh) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[j][h] = gelu_tanh2(v[j][h]);
        }
#pragma unroll
        for (int jp = 0; jp < 2; ++jp)
          stmatrix_x4(at(4 * g + 2 * jp), narrow(v[2 * jp][0]), narrow(v[2 * jp][1]), narrow(v[2 * jp + 1][0]),
                      narrow(v[2 * jp + 1][1]));
      }
    }
    __syncwarp();
    if (gated) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = warp * 16 + g4 + 8 * i;
        if (dst[i] != nullptr && n0 + tig * 16 < n_hi)
          *reinterpret_cast<uint4*>(dst[i] + n0 / 2) = lds128(sy + row * 128 + ((tig ^ (row & 7)) << 4));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = warp * 16 + (lane >> 3) + 4 * i;
        if (dst[i] != nullptr && n0 + ch * 8 < n_hi)
          *reinterpret_cast<uint4*>(dst[i] + n0) = lds128(sy + row * 128 + ((ch ^ (row & 7)) << 4));
      }
    }
    stage = stage + 1 == C::kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();
}

// ------------------------------------------------------------------ small
// Small batches: down and up of one 16-row tile in one launch.  What counts is
// the chain launch -> plan -> operands -> sum -> operands -> store, so it is
// made short: a cluster of eight CTAs shares the tile, each summing an eighth
// of the features (its warps straight from global memory into MMA fragments),
// the sums meet through distributed shared memory in rank order, and each CTA
// then writes its share of the columns, whose piece of P and Y it asked for
// before the first sum.  A sum over k may visit k in any order as long as both
// operands use the same one: thread tig of a quad takes the eight consecutive
// features 8 tig .. of every group of 32 (one 16-byte load per row), as k slots
// 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9 of two MMAs.
constexpr int kSmallCluster = 8;
template <int R>
struct SmallCfg {
  static constexpr int kStepCols = 256;  // 32 per warp
  static constexpr int kYStride = kStepCols * 2 + 16;  // bytes of a staged row of Y (conflict-free 4-byte reads)
  static constexpr int kOffY = R * kStepCols * 2;      // in a buffer: P's four pieces, then Y's 16 rows
  static constexpr int kBuf = kOffY + 16 * kYStride + 256;
  static constexpr int kBufs = R <= 16 ? 4 : R <= 64 ? 3 : 2;  // steps of P and Y, all but one asked for at the start
  static_assert(kBuf % 128 == 0, "P's pieces are 128-byte rows");
  static constexpr int kOffRed = kBufs * kBuf;              // 4 x [16][R] f32
  static constexpr int kOffSum = kOffRed + 4 * 16 * R * 4;  // [16][R] f32, read by the cluster
  static constexpr int kVStride = R * 2 + 16;              // bytes of a row of the bf16 hidden tile
  static constexpr int kOffV = kOffSum + 16 * R * 4;
  static constexpr int kSmemBytes = kOffV + 16 * kVStride;
  static constexpr int kMinCtas = 228 * 1024 / (kSmemBytes + 1024);  // per SM: 3, 2, 1, 1
};

struct SmallArgs {
  const __nv_bfloat16 *x, *y, *down, *up;
  const float* scale;
  const int32_t* words;
  __nv_bfloat16* out;
  __nv_bfloat16* hidden;  // [M, rank] or NULL
  float* hidden32;        // [M, rank] or NULL
  AdapterPlan lay;
  int64_t ldx, ldy, ldo;
  int K, N, rank, A, act, with_none, k_per_rank, cols_per_cta, ctas_per_tile;
};

template <int R>
__global__ void __launch_bounds__(256, SmallCfg<R>::kMinCtas) adapter_small_kernel(const SmallArgs a) {
  using C = SmallCfg<R>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  float* red = reinterpret_cast<float*>(smem_raw + C::kOffRed);
  const PlanTile t = plan_tile<kBlockRows>(a.words, a.lay, a.A, blockIdx.x / a.ctas_per_tile, a.with_none != 0);
  if (t.rows == 0) return;  // the whole cluster: it shares the tile
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, tig = lane & 3;
  const int part = blockIdx.x % a.ctas_per_tile;  // of the columns
  const int rank = part % kSmallCluster;          // in the cluster
  const bool none = t.adapter >= a.A;
  const int tok0 = a.words[a.lay.off_perm + t.row + g4];
  const int tok1 = a.words[a.lay.off_perm + t.row + g4 + 8];
  const int ytok0 = a.words[a.lay.off_perm + t.row + warp];
  const int ytok1 = a.words[a.lay.off_perm + t.row + warp + 8];
  const int n_lo = part * a.cols_per_cta;
  const int n_hi = min(a.N, n_lo + a.cols_per_cta);
  const __nv_bfloat16* U = none ? a.up : a.up + static_cast<int64_t>(t.adapter) * a.rank * a.N;

  // columns n0 .. n0 + 255 of P (four 64-column pieces of [R][128 bytes]) and of
  // the tile's rows of Y
  auto load_step = [&](int n0, int buf) {
    if (n0 < n_hi) {
      if (!none) {
#pragma unroll 4
        for (int c = tid; c < R * 32; c += 256) {
          const int row = c >> 5, cc = c & 31, col = n0 + cc * 8;
          const bool ok = row < a.rank && col < n_hi;
          cp_async_16(sbase + buf * C::kBuf + (cc >> 3) * (R * 128) + row * 128 + (((cc & 7) ^ (row & 7)) << 4),
                      ok ? U + static_cast<int64_t>(row) * a.N + col : a.up, ok);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // rows warp and warp + 8
        const int col = n0 + lane * 8;
        const int tok = i ? ytok1 : ytok0;
        if (tok >= 0 && col < n_hi)
          cp_async_16(sbase + buf * C::kBuf + C::kOffY + (warp + 8 * i) * C::kYStride + lane * 16,
                      a.y + static_cast<int64_t>(tok) * a.ldy + col, true);
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < C::kBufs - 1; ++i) load_step(n_lo + i * C::kStepCols, i);

  if (!none) {
    const __nv_bfloat16* x0 = a.x + static_cast<int64_t>(tok0) * a.ldx;
    const __nv_bfloat16* x1 = a.x + static_cast<int64_t>(tok1) * a.ldx;
    const __nv_bfloat16* P = a.down + static_cast<int64_t>(t.adapter) * a.rank * a.K;
    const int k_hi = min(a.K, (rank + 1) * a.k_per_rank);
    float acc[R / 8][4] = {};
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll (R <= 32 ? 2 : 1)
    for (int k = rank * a.k_per_rank + warp * 32 + tig * 8; k < k_hi + tig * 8; k += 256) {
      const bool in = k < k_hi;
      const uint4 u0 = in && tok0 >= 0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
      const uint4 u1 = in && tok1 >= 0 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
      uint4 p[R / 8];
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt)
        p[nt] = in && nt * 8 < a.rank ? ld_stream16(P + static_cast<int64_t>(nt * 8 + g4) * a.K + k) : zero;
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt) {
        mma_16816_bf16(acc[nt], u0.x, u1.x, u0.y, u1.y, p[nt].x, p[nt].y);
        mma_16816_bf16(acc[nt], u0.z, u1.z, u0.w, u1.w, p[nt].z, p[nt].w);
      }
    }
    // the eight warps' sums, in a fixed order: w + (w + 4), then over w
    auto at = [&](int w, int nt, int i) {
      return (w * 16 + g4 + 8 * (i >> 1)) * R + nt * 8 + 2 * tig + (i & 1);
    };
    if (warp >= 4) {
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[at(warp - 4, nt, i)] = acc[nt][i];
    }
    __syncthreads();
    if (warp < 4) {
#pragma unroll
      for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[at(warp, nt, i)] += acc[nt][i];
    }
    __syncthreads();
    for (int i = tid; i < 16 * R; i += 256)
      *reinterpret_cast<float*>(smem_raw + C::kOffSum + 4 * i) =
          (red[i] + red[16 * R + i]) + (red[32 * R + i] + red[48 * R + i]);
  }
  __syncwarp();
  cluster_sync();
  {
    const float s = none ? 0.f : a.scale[t.adapter];
    for (int i = tid; i < 16 * (R / 2); i += 256) {
      const int row = i / (R / 2), c = (i % (R / 2)) * 2;
      float2 v = make_float2(0.f, 0.f);
      // (columns past the rank are an infinite x times zeros: NaN, which would
      // meet the zeros of P's rows there)
      if (!none && c < a.rank) {
        float2 u[kSmallCluster];
#pragma unroll
        for (int q = 0; q < kSmallCluster; ++q)
          u[q] = ld_cluster_f2(mapa_shared(sbase + C::kOffSum + 4u * (row * R + c), q));
#pragma unroll
        for (int q = 0; q < kSmallCluster; ++q) {
          v.x += u[q].x;
          v.y += u[q].y;
        }
      }
      v.x *= s;
      v.y *= s;
      const uint32_t b = pack_bf16x2(v.x, v.y);
      sts32(sbase + C::kOffV + row * C::kVStride + 2 * c, b);
      if (part == 0 && a.hidden != nullptr && c < a.rank) {
        const int tok = a.words[a.lay.off_perm + t.row + row];
        if (tok >= 0) {
          const int64_t o = static_cast<int64_t>(tok) * a.rank + c;
          *reinterpret_cast<uint32_t*>(a.hidden + o) = b;
          if (a.hidden32 != nullptr) *reinterpret_cast<float2*>(a.hidden32 + o) = v;
        }
      }
    }
  }
  __syncwarp();
  cluster_arrive();  // this CTA has read the others' sums

  int buf = 0;
  for (int n0 = n_lo; n0 < n_hi; n0 += C::kStepCols, buf = buf + 1 == C::kBufs ? 0 : buf + 1) {
    cp_async_wait<C::kBufs - 2>();
    __syncthreads();  // P of this step and the hidden tile are there; the last step's buffer is free
    load_step(n0 + (C::kBufs - 1) * C::kStepCols, buf == 0 ? C::kBufs - 1 : buf - 1);
    float acc[4][4] = {};
    if (!none) {
      const int wcol = warp * 32;
      const uint32_t piece = sbase + buf * C::kBuf + (wcol / 64) * (R * 128);
      const int krow = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int ks = 0; ks < R / 16; ++ks) {
        uint32_t af[4];
        ldmatrix_x4(sbase + C::kOffV + (lane & 15) * C::kVStride + (2 * ks + (lane >> 4)) * 16, af);
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
          uint32_t bf[4];
          const int row = ks * 16 + krow;
          const int ch = (wcol % 64) / 8 + 2 * jp + (lane >> 4);
          ldmatrix_x4_trans(piece + row * 128 + ((ch ^ (row & 7)) << 4), bf);
          mma_16816_bf16(acc[2 * jp], af[0], af[1], af[2], af[3], bf[0], bf[1]);
          mma_16816_bf16(acc[2 * jp + 1], af[0], af[1], af[2], af[3], bf[2], bf[3]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int tok = h ? tok1 : tok0;
      F2 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = add2(widen(lds32(sbase + buf * C::kBuf + C::kOffY + (g4 + 8 * h) * C::kYStride +
                                (warp * 32 + 8 * j + 2 * tig) * 2)),
                    f2(acc[j][2 * h], acc[j][2 * h + 1]));
      const int col = n0 + warp * 32 + 2 * tig;
      if (a.act == kActGeluTanh) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = gelu_tanh2(v[j]);
      } else if (a.act != kActNone) {  // n-tiles 0, 1 hold 16 gate columns, 2, 3 their up columns
        v[0] = mul2(gate2(v[0], a.act), v[2]);
        v[1] = mul2(gate2(v[1], a.act), v[3]);
      }
      if (tok < 0) continue;
      if (a.act == kActNone || a.act == kActGeluTanh) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (col + 8 * j < n_hi)
            *reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(tok) * a.ldo + col + 8 * j) = narrow(v[j]);
      } else if (col < n_hi) {
        const int oc = (n0 + warp * 32) / 2 + 2 * tig;
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<uint32_t*>(a.out + static_cast<int64_t>(tok) * a.ldo + oc + 8 * j) = narrow(v[j]);
      }
    }
  }
  cp_async_wait<0>();
  __syncwarp();
  cluster_wait();  // the others have read this CTA's sums
}

// ------------------------------------------------------------------ wgrad
// dP_a[r, c] = sum over a's rows of G[m, r] X[m, c], as D = X^T G on tcgen05:
// M = 128 columns of X, N = R, k = tokens, both operands MN-major (a token's
// features are contiguous) in 128-byte-swizzled [64 tokens][64 features]
// blocks.  D's lanes are columns of dP, so its rows leave tensor memory
// coalesced, without a transpose.  (Warp-level MMAs with ldmatrix.trans
// fragments ran the same sums at 1.7 TB/s of X.)  Measured: X of 4608 x 12288
// at r = 64 in a loop of 20 us, 5.7 TB/s; 8-bit X of 4608 x 4096 15 us.
//
// CTA = (column tile, row split): the plan's rows are cut into splits of L rows
// whatever the adapters; a CTA walks its rows in stages of 64 and changes to
// its other accumulator at each adapter's end, while four warps write the
// finished one: straight to the bf16 result if the split holds all of the
// adapter's rows, else to one of the split's two f32 slots: 0 for the adapter
// that began in an earlier split, 1 for the one that goes on in a later one
// (there is at most one of each).  A reduce kernel adds an adapter's slots in
// order.  No atomics.
//
// An 8-bit X: the codes go through a ring of their own (each thread converts
// the 16 bytes it copied itself), become bf16 exactly ((128 + low seven bits)
// - (128 or 256)), and the row's scale of this 128-column tile multiplies G
// instead, in f32, rounded once to bf16 as the MMA's operand.
template <int R, bool I8>
struct WgradCfg {
  static constexpr int kCols = 128;
  static constexpr int kRows = 64;
  static constexpr int kBlock = kRows * 128;            // [64 tokens][64 features] bf16
  static constexpr int kGBlocks = (R + 63) / 64;
  static constexpr int kStage = (2 + kGBlocks) * kBlock;
  static constexpr int kStages = I8 ? 3 : (R <= 64 ? 4 : 3);
  static constexpr int kAhead = I8 ? 0 : kStages - 2;   // stages a thread's copies run ahead
  static constexpr int kRaw = I8 ? 4 : 0;               // stages of raw codes
  static constexpr int kRawStage = kRows * 128;
  static constexpr int kThreads = (4 + 1 + 8) * 32;     // epilogue, MMA, producer warps
  static constexpr int kOffRaw = kStages * kStage;
  static constexpr int kOffBar = kOffRaw + kRaw * kRawStage;
  static constexpr int kSmemBytes = kOffBar + 16 * kStages + 64 + 1024;
  static constexpr int kMinCtas = 2 * (kSmemBytes + 1024) <= 228 * 1024 ? 2 : 1;
  static constexpr int kTmemCols = 2 * R;
};

// One weight gradient: X [M, cols] with its scales if it is in 8 bits, G [M, rank]
// (g32 with an 8-bit X), the partial sums and the result.
struct WgradProblem {
  const void* x;
  const float* x_scales;
  const __nv_bfloat16* g;
  const float* g32;
  float* part;
  __nv_bfloat16* dbank;
  int64_t ldx;
  int cols, col_tiles, rows_per_split;
};
// One launch computes one or two of them: CTAs past the first's column tiles
// take the second.
struct WgradArgs {
  WgradProblem first, second;
  const int32_t* words;
  unsigned int* error;
  AdapterPlan lay;
  int rank, A;
  int alone;  // one split and few adapters: no reduce kernel follows
};

// Four int8 codes -> two bf16 pairs, exact.
__device__ __forceinline__ void i8_to_bf16(uint32_t u, uint32_t& p01, uint32_t& p23) {
  const uint32_t low = u & 0x7F7F7F7Fu, sign = u & 0x80808080u;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p01) : "r"(prmt(low, 0x43u, 0x4140u)), "r"(prmt(sign, 0x43u, 0x4140u)));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(p23) : "r"(prmt(low, 0x43u, 0x4342u)), "r"(prmt(sign, 0x43u, 0x4342u)));
}

// Rows of a split in stages of 64 that never cross an adapter's end.
struct RowCursor {
  const int32_t* blk;
  const int32_t* starts;
  int pos, end, hi, adapter;
  __device__ __forceinline__ RowCursor(const int32_t* words, const AdapterPlan& lay, int lo, int hi_)
      : blk(words + lay.off_blk), starts(words + lay.off_start), pos(lo), end(lo), hi(hi_), adapter(0) {
    open();
  }
  __device__ __forceinline__ bool live() const { return pos < hi; }
  __device__ __forceinline__ void open() {
    if (pos < hi) {
      adapter = blk[pos / 16];
      end = min(hi, starts[adapter + 1]);
    }
  }
  // to the next stage; true if the adapter's rows of this split are done
  __device__ __forceinline__ bool next() {
    pos += 64;
    if (pos < end) return false;
    pos = end;
    open();
    return true;
  }
};

template <int R, bool I8>
__global__ void __launch_bounds__(WgradCfg<R, I8>::kThreads, WgradCfg<R, I8>::kMinCtas)
    adapter_wgrad_kernel(const WgradArgs a) {
  using C = WgradCfg<R, I8>;
  const bool second = static_cast<int>(blockIdx.x) >= a.first.col_tiles;
  const WgradProblem w = second ? a.second : a.first;
  const int col_tile = blockIdx.x - (second ? a.first.col_tiles : 0);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t sbase = (raw + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (sbase - raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto full_bar = [&](int s) { return sbase + C::kOffBar + 8u * s; };
  auto empty_bar = [&](int s) { return sbase + C::kOffBar + 8u * (C::kStages + s); };
  auto acc_full = [&](int b) { return sbase + C::kOffBar + 16u * C::kStages + 8u * b; };
  auto acc_empty = [&](int b) { return sbase + C::kOffBar + 16u * C::kStages + 16u + 8u * b; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kOffBar + 16 * C::kStages + 32);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffBar + 16 * C::kStages + 40);
  if (tid == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full_bar(s), 8);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full(b), 1);
      mbar_init(acc_empty(b), 4);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 4) {
    tmem_alloc(smem_u32(tmem_slot), C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int col0 = col_tile * C::kCols;
  const int row_lo = blockIdx.y * w.rows_per_split;  // (past the rows: no work)
  const int row_hi = min(row_lo + w.rows_per_split, a.words[AdapterPlan::kNoneStart]);
  grid_wait();  // G may be the output of the kernel before this one
  RowCursor cur(a.words, a.lay, row_lo, row_hi);

  if (warp >= 5) {
    // -------------------------------------------------------------- producers
    const int32_t* perm = a.words + a.lay.off_perm;
    const int pt = tid - 160;
    if constexpr (!I8) {
      const int ch = pt & 15;  // 16-byte chunk of a row's 128 columns
      const bool col_ok = col0 + ch * 8 < w.cols;
      const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(w.x) + col0 + ch * 8;
      // the tokens of a stage's rows, looked up one stage ahead
      constexpr int kG = (64 * (R / 8) + 255) / 256;
      int tx[4], tg[kG];
      auto look_up = [&]() {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (pt >> 4) + 16 * i;
          tx[i] = cur.live() && cur.pos + row < cur.end ? perm[cur.pos + row] : -1;
        }
#pragma unroll
        for (int i = 0; i < kG; ++i) {
          const int row = (pt + 256 * i) / (R / 8);
          tg[i] = cur.live() && row < 64 && cur.pos + row < cur.end ? perm[cur.pos + row] : -1;
        }
      };
      look_up();
      int it = 0;
      for (; cur.live(); ++it) {
        const int slot = it % C::kStages;
        if (!mbar_wait(empty_bar(slot), static_cast<uint32_t>(((it / C::kStages) & 1) ^ 1), abort_flag)) break;
        const uint32_t sx = sbase + slot * C::kStage, sg = sx + 2 * C::kBlock;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = (pt >> 4) + 16 * i;
          const bool ok = tx[i] >= 0 && col_ok;
          cp_async_16_l2(sx + (ch >> 3) * C::kBlock + row * 128 + (((ch & 7) ^ (row & 7)) << 4),
                         ok ? x + static_cast<int64_t>(tx[i]) * w.ldx : static_cast<const __nv_bfloat16*>(w.x), ok);
        }
#pragma unroll
        for (int i = 0; i < kG; ++i) {
          const int e = pt + 256 * i;
          const int row = e / (R / 8), gc = e % (R / 8);
          if (64 * (R / 8) % 256 != 0 && row >= 64) break;
          const bool ok = tg[i] >= 0 && gc * 8 < a.rank;
          cp_async_16(sg + (gc >> 3) * C::kBlock + row * 128 + (((gc & 7) ^ (row & 7)) << 4),
                      ok ? w.g + static_cast<int64_t>(tg[i]) * a.rank + gc * 8 : w.g, ok);
        }
        cp_async_commit();
        cur.next();
        look_up();
        if (it >= C::kAhead) {
          cp_async_wait<C::kAhead>();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(full_bar((it - C::kAhead) % C::kStages));
        }
      }
      cp_async_wait<0>();
      fence_proxy_async_smem();
      __syncwarp();
      if (!cur.live() && lane == 0)
        for (int s = max(0, it - C::kAhead); s < it; ++s) mbar_arrive(full_bar(s % C::kStages));
    } else {
      const int8_t* x = static_cast<const int8_t*>(w.x);
      const int ncb = (w.cols + 127) / 128;
      const int ch = pt & 7;  // 16 codes
      const bool col_ok = col0 + ch * 16 < w.cols;
      RowCursor rc(a.words, a.lay, row_lo, row_hi);  // raw codes, kRaw stages ahead
      int rit = 0;
      int tx[2];  // tokens of the next stage's rows, looked up one stage ahead
      auto look_raw = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = (pt >> 3) + 32 * i;
          tx[i] = rc.live() && rc.pos + row < rc.end ? perm[rc.pos + row] : -1;
        }
      };
      look_raw();
      auto load_raw = [&]() {
        if (rc.live()) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int token = tx[i];
            const bool ok = token >= 0 && col_ok;
            cp_async_16(sbase + C::kOffRaw + (rit % C::kRaw) * C::kRawStage + (pt + 256 * i) * 16,
                        ok ? x + static_cast<int64_t>(token) * w.ldx + col0 + ch * 16 : x, ok);
          }
          rc.next();
          ++rit;
          look_raw();
        }
        cp_async_commit();
      };
      // G: four threads per row, R / 4 values each, one stage ahead
      RowCursor gc(a.words, a.lay, row_lo, row_hi);
      const int grow = pt >> 2, g0 = (pt & 3) * (R / 4);
      float4 gv[R / 16];
      float gs = 0.f;
      int tg = gc.live() && gc.pos + grow < gc.end ? perm[gc.pos + grow] : -1;
      auto load_g = [&]() {
        gs = 0.f;
#pragma unroll
        for (int i = 0; i < R / 16; ++i) gv[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (gc.live()) {
          const int token = tg;
          if (token >= 0) {
            gs = __ldg(w.x_scales + static_cast<int64_t>(token) * ncb + col_tile);
#pragma unroll
            for (int i = 0; i < R / 16; ++i)
              if (g0 + 4 * i < a.rank)
                gv[i] = __ldg(reinterpret_cast<const float4*>(w.g32 + static_cast<int64_t>(token) * a.rank + g0 + 4 * i));
          }
          gc.next();
          tg = gc.live() && gc.pos + grow < gc.end ? perm[gc.pos + grow] : -1;
        }
      };
#pragma unroll
      for (int i = 0; i < C::kRaw - 1; ++i) load_raw();
      load_g();
      int it = 0;
      for (; cur.live(); ++it) {
        const int slot = it % C::kStages;
        load_raw();
        cp_async_wait<C::kRaw - 1>();
        uint4 codes[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          codes[i] = lds128(sbase + C::kOffRaw + (it % C::kRaw) * C::kRawStage + (pt + 256 * i) * 16);
        if (!mbar_wait(empty_bar(slot), static_cast<uint32_t>(((it / C::kStages) & 1) ^ 1), abort_flag)) break;
        const uint32_t sx = sbase + slot * C::kStage, sg = sx + 2 * C::kBlock;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = (pt >> 3) + 32 * i;
          const uint32_t c4[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
          uint32_t o[8];
#pragma unroll
          for (int q = 0; q < 4; ++q) i8_to_bf16(c4[q], o[2 * q], o[2 * q + 1]);
          const uint32_t base = sx + (ch >> 2) * C::kBlock + row * 128;
          const int c0 = (ch & 3) * 2;
          sts128(base + ((c0 ^ (row & 7)) << 4), make_uint4(o[0], o[1], o[2], o[3]));
          sts128(base + (((c0 + 1) ^ (row & 7)) << 4), make_uint4(o[4], o[5], o[6], o[7]));
        }
#pragma unroll
        for (int i = 0; i < R / 16; ++i) {
          const int c = g0 + 4 * i;  // 8 bytes: half a chunk
          const uint32_t at = sg + (c >> 6) * C::kBlock + grow * 128 + ((((c & 63) >> 3) ^ (grow & 7)) << 4) + (c & 4) * 2;
          sts64(at, pack_bf16x2(gv[i].x * gs, gv[i].y * gs), pack_bf16x2(gv[i].z * gs, gv[i].w * gs));
        }
        load_g();
        cur.next();
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(full_bar(slot));
      }
      cp_async_wait<0>();
    }
  } else if (warp == 4) {
    // ------------------------------------------------------------------- MMA
    constexpr uint32_t idesc = make_idesc_bf16(128, R) | (1u << 15) | (1u << 16);  // both operands MN-major
    int it = 0, seg = 0;
    bool fresh = true;
    while (cur.live()) {
      const int slot = it % C::kStages, b = seg & 1;
      if (fresh && !mbar_wait(acc_empty(b), static_cast<uint32_t>(((seg >> 1) & 1) ^ 1), abort_flag)) break;
      if (!mbar_wait(full_bar(slot), static_cast<uint32_t>((it / C::kStages) & 1), abort_flag)) break;
      tc_fence_after();
      const uint64_t ad = make_sw128_mnmajor_desc(sbase + slot * C::kStage, C::kBlock);
      const uint64_t bd = make_sw128_mnmajor_desc(sbase + slot * C::kStage + 2 * C::kBlock, C::kBlock);
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)  // 16 tokens: two 8-row groups, 2048 bytes
        tc_mma_ss_elect(tmem + b * R, ad + 128 * ks, bd + 128 * ks, idesc, !(fresh && ks == 0));
      tc_commit_elect(empty_bar(slot));
      ++it;
      fresh = cur.next();
      if (fresh) {
        tc_commit_elect(acc_full(b));
        ++seg;
      }
    }
    __syncwarp();
  } else {
    // -------------------------------------------------------------- epilogue
    const int32_t* starts = a.words + a.lay.off_start;
    const int col = col0 + 32 * warp + lane;
    for (int seg = 0; cur.live(); ++seg) {
      const int b = seg & 1, ad = cur.adapter;
      if (!mbar_wait(acc_full(b), static_cast<uint32_t>((seg >> 1) & 1), abort_flag)) break;
      tc_fence_after();
      const bool whole = starts[ad] >= row_lo && starts[ad + 1] <= row_lo + w.rows_per_split;
      const int64_t slot = whole ? ad : 2 * static_cast<int>(blockIdx.y) + (starts[ad] < row_lo ? 0 : 1);
      const int64_t base = slot * a.rank * w.cols + col;
#pragma unroll 1
      for (int c = 0; c < R; c += 16) {
        uint32_t v[16];
        tmem_ld_x16(tmem + (static_cast<uint32_t>(32 * warp) << 16) + b * R + c, v);
        tmem_wait_ld();
        if (col < w.cols) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            if (c + (e & 8) >= a.rank) break;
            const int64_t o = base + static_cast<int64_t>(c + e) * w.cols;
            if (whole)
              w.dbank[o] = __float2bfloat16_rn(__uint_as_float(v[e]));
            else
              w.part[o] = __uint_as_float(v[e]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(b));
      cur.pos = cur.end;
      cur.open();
    }
    if (a.alone && col < w.cols) {  // zeros for adapters without rows
      for (int ad = 0; ad < a.A; ++ad)
        if (starts[ad] == starts[ad + 1])
          for (int r = 0; r < a.rank; ++r)
            w.dbank[(static_cast<int64_t>(ad) * a.rank + r) * w.cols + col] = __float2bfloat16_rn(0.f);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort_flag) atomicOr(a.error, 1u << kErrTimeout);
  if (warp == 4) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Adds the slots of adapters that several splits share, in split order; zeros
// for adapters without rows.  blockIdx.y: adapter; z: problem.
__global__ void __launch_bounds__(256) adapter_wgrad_reduce_kernel(const WgradArgs a) {
  const WgradProblem w = blockIdx.z == 0 ? a.first : a.second;
  const int64_t elems = static_cast<int64_t>(a.rank) * w.cols;
  const int ad = blockIdx.y;
  const int lo = a.words[a.lay.off_start + ad], hi = a.words[a.lay.off_start + ad + 1];
  grid_wait();
  const int s0 = lo / w.rows_per_split, s1 = hi > lo ? (hi - 1) / w.rows_per_split : s0;
  if (hi > lo && s0 == s1) return;
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < elems; i += gridDim.x * 1024ll) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (hi > lo)
      for (int s = s0; s <= s1; ++s) {
        const float4 u =
            __ldcg(reinterpret_cast<const float4*>(w.part + static_cast<int64_t>(2 * s + (s == s0 ? 1 : 0)) * elems + i));
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
    *reinterpret_cast<uint2*>(w.dbank + static_cast<int64_t>(ad) * elems + i) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
}

}  // namespace dq
