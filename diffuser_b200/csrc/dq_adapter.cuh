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
// 64 FLOP/B at r = 64, against the machine's 256.  Hence warp-level bf16 MMAs
// with operands from shared memory, and everything is arranged around the
// stream of the wide operand: each element of it is read once per kernel, in
// 16-byte pieces, several stages ahead.
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
#include "dq_ptx.cuh"
#include "dq_smallm.cuh"

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
  p.off_blk = p.off_perm + p.cap;
  p.off_tiles = p.off_blk + up4(p.cap / 16);
  p.words = p.off_tiles + up4(p.max_tiles);
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
  if ((bad || bad_id) && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(error, 1u << 10);
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
  for (int i = lane; i < tiles; i += 32) words[lay.off_tiles + tile0 + i] = row0 + i * kTileRows;
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
};
template <int T>
__device__ __forceinline__ PlanTile plan_tile(const int32_t* words, const AdapterPlan& lay, int A,
                                              int tile, bool with_none) {
  PlanTile t{0, 0, A};
  if constexpr (T == kTileRows) {
    if (tile >= words[with_none ? AdapterPlan::kAllTiles : AdapterPlan::kTiles]) return t;
    t.row = words[lay.off_tiles + tile];
    t.adapter = words[lay.off_blk + t.row / 16];
    t.rows = min(T, words[lay.off_start + t.adapter + 1] - t.row);
  } else {
    t.row = tile * T;
    if (t.row >= words[with_none ? AdapterPlan::kRows : AdapterPlan::kNoneStart]) return t;
    t.adapter = words[lay.off_blk + tile];
    t.rows = T;
  }
  return t;
}

// ------------------------------------------------------------- small wrappers
// 16-byte asynchronous copy; with `ok` false the destination is zero-filled
// and nothing is read.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_4z(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// ------------------------------------------------------------------- down
// part[split][row][r] = sum over the split's k of X[perm[row]][k] P_a[r][k],
// f32; the reader adds the splits in order.
//
// Large tiles (128 rows, one warp per 16): X and P move through a cp.async
// ring of 64-feature stages (128-byte rows, 16-byte chunk c of row i at
// c ^ (i % 8): conflict-free for the copies and for ldmatrix).
template <int R>
struct DownCfg {
  static constexpr int kStageX = kTileRows * 128;
  static constexpr int kStageP = R * 128;
  static constexpr int kStages = R <= 64 ? 4 : 3;
  static constexpr int kSmemBytes = kStages * (kStageX + kStageP);
};

struct DownArgs {
  const __nv_bfloat16* x;
  const __nv_bfloat16* bank;
  const int32_t* words;
  float* part;
  AdapterPlan lay;
  int64_t ldx;
  int K, rank, A, k_per_split;
};

template <int R>
__global__ void __launch_bounds__(256, 2) adapter_down_kernel(const DownArgs a) {
  using C = DownCfg<R>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const PlanTile t = plan_tile<kTileRows>(a.words, a.lay, a.A, blockIdx.x, false);
  grid_launch_dependents();
  if (t.rows == 0) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int k_lo = blockIdx.y * a.k_per_split;
  const int k_hi = min(a.K, k_lo + a.k_per_split);
  const int steps = (k_hi - k_lo + 63) / 64;
  const __nv_bfloat16* P = a.bank + static_cast<int64_t>(t.adapter) * a.rank * a.K;

  // this thread copies chunk tid % 8 of rows tid / 8 + 32 i
  const int chunk = tid & 7;
  const __nv_bfloat16* src[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (tid >> 3) + 32 * i;
    const int token = row < t.rows ? a.words[a.lay.off_perm + t.row + row] : -1;
    src[i] = token >= 0 ? a.x + static_cast<int64_t>(token) * a.ldx : nullptr;
  }
  auto load = [&](int step) {
    if (step < steps) {
      const uint32_t sx = sbase + (step % C::kStages) * (C::kStageX + C::kStageP);
      const uint32_t sp = sx + C::kStageX;
      const int k = k_lo + step * 64 + chunk * 8;
      const bool in = k < k_hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = (tid >> 3) + 32 * i;
        const bool ok = in && src[i] != nullptr;
        cp_async_16(sx + row * 128 + ((chunk ^ (row & 7)) << 4), ok ? src[i] + k : a.x, ok);
      }
#pragma unroll
      for (int i = 0; i < (R * 8 + 255) / 256; ++i) {
        const int row = (tid >> 3) + 32 * i;
        const bool ok = in && row < a.rank;
        if (row < R)
          cp_async_16(sp + row * 128 + ((chunk ^ (row & 7)) << 4),
                      ok ? P + static_cast<int64_t>(row) * a.K + k : a.bank, ok);
      }
    }
    cp_async_commit();
  };

  float acc[R / 8][4] = {};
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) load(s);
  const bool active = warp * 16 < t.rows;
  for (int step = 0; step < steps; ++step) {
    cp_async_wait<C::kStages - 2>();
    __syncthreads();
    load(step + C::kStages - 1);
    if (!active) continue;
    const uint32_t sx = sbase + (step % C::kStages) * (C::kStageX + C::kStageP);
    const uint32_t sp = sx + C::kStageX;
    const int arow = warp * 16 + (lane & 15);
    const int brow = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      uint32_t af[4];
      ldmatrix_x4(sx + arow * 128 + (((2 * ks + (lane >> 4)) ^ (arow & 7)) << 4), af);
#pragma unroll
      for (int nt = 0; nt < R / 16; ++nt) {
        uint32_t bf[4];
        const int row = nt * 16 + brow;
        ldmatrix_x4(sp + row * 128 + (((2 * ks + ((lane >> 3) & 1)) ^ (row & 7)) << 4), bf);
        mma_16816_bf16(acc[2 * nt], af[0], af[1], af[2], af[3], bf[0], bf[1]);
        mma_16816_bf16(acc[2 * nt + 1], af[0], af[1], af[2], af[3], bf[2], bf[3]);
      }
    }
  }
  if (!active) return;
  float* out = a.part + (static_cast<int64_t>(blockIdx.y) * a.lay.cap + t.row + warp * 16) * a.rank;
  const int g4 = lane >> 2, tig = lane & 3;
#pragma unroll
  for (int nt = 0; nt < R / 8; ++nt)
    if (nt * 8 < a.rank) {
      const int c = nt * 8 + 2 * tig;
      *reinterpret_cast<float2*>(out + static_cast<int64_t>(g4) * a.rank + c) = make_float2(acc[nt][0], acc[nt][1]);
      *reinterpret_cast<float2*>(out + static_cast<int64_t>(g4 + 8) * a.rank + c) =
          make_float2(acc[nt][2], acc[nt][3]);
    }
}

// Small tiles (16 rows): the latency of the chain launch -> plan -> operands
// -> sum is what counts, so the warps of a CTA share the split's k between
// them and load straight into MMA fragments.  A sum over k may visit k in any
// order as long as both operands use the same one: thread tig of a quad takes
// the eight consecutive features 8 tig .. of every group of 32 (one 16-byte
// load per row), as k slots 2 tig, 2 tig + 1, 2 tig + 8, 2 tig + 9 of two MMAs.
template <int R>
__global__ void __launch_bounds__(256) adapter_down_small_kernel(const DownArgs a) {
  __shared__ float red[4][16 * R];
  const PlanTile t = plan_tile<kBlockRows>(a.words, a.lay, a.A, blockIdx.x, false);
  grid_launch_dependents();
  if (t.rows == 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g4 = lane >> 2, tig = lane & 3;
  const int t0 = a.words[a.lay.off_perm + t.row + g4];
  const int t1 = a.words[a.lay.off_perm + t.row + g4 + 8];
  const __nv_bfloat16* x0 = a.x + static_cast<int64_t>(t0) * a.ldx;
  const __nv_bfloat16* x1 = a.x + static_cast<int64_t>(t1) * a.ldx;
  const __nv_bfloat16* P = a.bank + static_cast<int64_t>(t.adapter) * a.rank * a.K;
  const int k_hi = min(a.K, static_cast<int>(blockIdx.y + 1) * a.k_per_split);
  float acc[R / 8][4] = {};
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll (R <= 32 ? 2 : 1)
  for (int k = blockIdx.y * a.k_per_split + warp * 32 + tig * 8; k < k_hi + tig * 8; k += 256) {
    const bool in = k < k_hi;
    const uint4 u0 = in && t0 >= 0 ? *reinterpret_cast<const uint4*>(x0 + k) : zero;
    const uint4 u1 = in && t1 >= 0 ? *reinterpret_cast<const uint4*>(x1 + k) : zero;
    uint4 p[R / 8];
#pragma unroll
    for (int nt = 0; nt < R / 8; ++nt)
      p[nt] = in && nt * 8 < a.rank
                  ? ld_stream16(P + static_cast<int64_t>(nt * 8 + g4) * a.K + k)
                  : zero;
#pragma unroll
    for (int nt = 0; nt < R / 8; ++nt) {
      mma_16816_bf16(acc[nt], u0.x, u1.x, u0.y, u1.y, p[nt].x, p[nt].y);
      mma_16816_bf16(acc[nt], u0.z, u1.z, u0.w, u1.w, p[nt].z, p[nt].w);
    }
  }
  // the eight warps' sums, in a fixed order: w + (w + 4), then over w
  auto at = [&](int nt, int i) { return (g4 + 8 * (i >> 1)) * R + nt * 8 + 2 * tig + (i & 1); };
  if (warp >= 4) {
#pragma unroll
    for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[warp - 4][at(nt, i)] = acc[nt][i];
  }
  __syncthreads();
  if (warp < 4) {
#pragma unroll
    for (int nt = 0; nt < R / 8; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[warp][at(nt, i)] += acc[nt][i];
  }
  __syncthreads();
  float* out = a.part + (static_cast<int64_t>(blockIdx.y) * a.lay.cap + t.row) * a.rank;
  for (int i = threadIdx.x; i < 16 * R; i += 256) {
    const int row = i / R, c = i - row * R;
    if (c < a.rank) out[row * a.rank + c] = (red[0][i] + red[1][i]) + (red[2][i] + red[3][i]);
  }
}

// --------------------------------------------------------------------- up
// O[m, :] = act(Y[m, :] + s_a v[m, :] . P_a), v the sum of the down kernel's
// splits, rounded to bf16 here, once, for the MMA (its 2^-9 is on the added
// term alone; O is rounded to bf16 after the add).
//
// A warp owns 16 rows and CW columns at a time.  P's 64-column pieces are
// staged in shared memory with their columns permuted: 4-byte pair j of the
// 16-byte chunk t of a 32-column group is stored as pair t of chunk j, so that
// MMA column 2 tig + e of n-tile j is column 8 tig + 2 j + e of the group and
// each thread's accumulators are 16 consecutive bytes of a row of O: Y is read
// and O written in 16-byte pieces without another trip through shared memory.
template <int R, int WM>
struct UpCfg {
  static constexpr int kRows = 16 * WM;
  static constexpr int WN = 8 / WM;
  static constexpr int kWarpCols = WM == 8 ? 64 : 32;
  static constexpr int kStepCols = WN * kWarpCols;  // 64 or 256
  static constexpr int kGroups = kWarpCols / 32;
  static constexpr int kChunks = R * kStepCols / 8;          // 16-byte pieces of P per step
  static constexpr int kPerThread = (kChunks + 255) / 256;
  static constexpr int kBuf = R * kStepCols * 2;
  static constexpr int kBufs = WM == 8 ? 2 : 1;
  static constexpr int kSmemBytes = kBufs * kBuf;
};

struct UpArgs {
  const __nv_bfloat16* y;
  const __nv_bfloat16* bank;
  const float* scale;
  const int32_t* words;
  const float* part;
  __nv_bfloat16* out;
  __nv_bfloat16* hidden;
  AdapterPlan lay;
  int64_t ldy, ldo;
  int N, rank, A, splits, act, with_none, cols_per_cta;
};

__device__ __forceinline__ void unpack8(uint4 u, float* v) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}

template <int R, int WM>
__global__ void __launch_bounds__(256, 2) adapter_up_kernel(const UpArgs a) {
  using C = UpCfg<R, WM>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  const PlanTile t = plan_tile<C::kRows>(a.words, a.lay, a.A, blockIdx.x, a.with_none != 0);
  if (t.rows == 0) {
    grid_wait();  // no CTA ends before the grid it depends on
    return;
  }
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, tig = lane & 3;
  const int wm = warp % WM, wn = warp / WM;
  const int n_lo = blockIdx.y * a.cols_per_cta;
  const int n_hi = min(a.N, n_lo + a.cols_per_cta);
  const bool none = t.adapter >= a.A;
  const bool active = wm * 16 < t.rows;
  const int tok0 = active ? a.words[a.lay.off_perm + t.row + wm * 16 + g4] : -1;
  const int tok1 = active ? a.words[a.lay.off_perm + t.row + wm * 16 + g4 + 8] : -1;
  const __nv_bfloat16* P = none ? a.bank : a.bank + static_cast<int64_t>(t.adapter) * a.rank * a.N;
  const bool gated = act_is_gated(a.act);

  uint4 preg[C::kPerThread];
  auto load_p = [&](int n0) {
#pragma unroll
    for (int i = 0; i < C::kPerThread; ++i) {
      const int c = tid + 256 * i;
      const int row = c / (C::kStepCols / 8), col = n0 + (c % (C::kStepCols / 8)) * 8;
      const bool ok = !none && row < a.rank && col < n_hi && c < C::kChunks;
      preg[i] = ok ? __ldg(reinterpret_cast<const uint4*>(P + static_cast<int64_t>(row) * a.N + col))
                   : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  auto store_p = [&](int buf) {
#pragma unroll
    for (int i = 0; i < C::kPerThread; ++i) {
      const int c = tid + 256 * i;
      if (C::kChunks % 256 != 0 && c >= C::kChunks) break;
      const int row = c / (C::kStepCols / 8), cc = c % (C::kStepCols / 8);
      // 64-column piece cc / 8, 32-column group (cc / 4) % 2, chunk cc % 4
      const uint32_t base = sbase + buf * C::kBuf + (cc >> 3) * (R * 128) + row * 128 + 4 * (cc & 3);
      const uint32_t w[4] = {preg[i].x, preg[i].y, preg[i].z, preg[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sts32(base + (((((cc >> 2) & 1) * 4 + j) ^ (row & 7)) << 4), w[j]);
    }
  };
  // this thread's 8 columns of each 32-column group of its two rows
  uint4 yreg[C::kGroups][2];
  auto load_y = [&](int n0) {
#pragma unroll
    for (int g = 0; g < C::kGroups; ++g) {
      const int col = n0 + wn * C::kWarpCols + g * 32 + 8 * tig;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tok = h ? tok1 : tok0;
        if (tok >= 0 && col < n_hi)
          yreg[g][h] = *reinterpret_cast<const uint4*>(a.y + static_cast<int64_t>(tok) * a.ldy + col);
      }
    }
  };
  load_p(n_lo);
  load_y(n_lo);

  // the down kernel's sums
  grid_wait();
  uint32_t vf[R / 16][4];
  {
    const float s = none ? 0.f : a.scale[t.adapter];
    const int64_t split_stride = a.lay.cap * a.rank;
    const float* base = a.part + static_cast<int64_t>(t.row + wm * 16 + g4) * a.rank + 2 * tig;
#pragma unroll
    for (int ks = 0; ks < R / 16; ++ks)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int c = ks * 16 + 8 * (q >> 1);
        float2 v = make_float2(0.f, 0.f);
        if (!none && active && c < a.rank) {
          const float* p = base + static_cast<int64_t>(8 * (q & 1)) * a.rank + c;
          for (int i = 0; i < a.splits; ++i) {
            const float2 u = __ldcg(reinterpret_cast<const float2*>(p + i * split_stride));
            v.x += u.x;
            v.y += u.y;
          }
        }
        vf[ks][q] = pack_bf16x2(v.x * s, v.y * s);
        if (a.hidden != nullptr && blockIdx.y == 0 && wn == 0 && c < a.rank) {
          const int tok = (q & 1) ? tok1 : tok0;
          if (tok >= 0)
            *reinterpret_cast<uint32_t*>(a.hidden + static_cast<int64_t>(tok) * a.rank + c + 2 * tig) = vf[ks][q];
        }
      }
  }
  grid_launch_dependents();
  store_p(0);
  __syncthreads();

  int buf = 0;
  for (int n0 = n_lo; n0 < n_hi; n0 += C::kStepCols) {
    uint4 ycur[C::kGroups][2];
#pragma unroll
    for (int g = 0; g < C::kGroups; ++g) {
      ycur[g][0] = yreg[g][0];
      ycur[g][1] = yreg[g][1];
    }
    const bool more = n0 + C::kStepCols < n_hi;
    if (more) {
      load_p(n0 + C::kStepCols);
      load_y(n0 + C::kStepCols);
    }
    float acc[C::kGroups][4][4] = {};
    if (!none && active) {
      const int wcol = wn * C::kWarpCols;
      const uint32_t piece = sbase + buf * C::kBuf + (wcol / 64) * (R * 128);
      const int g0 = (wcol % 64) / 32;
      const int krow = (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
      for (int ks = 0; ks < R / 16; ++ks)
#pragma unroll
        for (int g = 0; g < C::kGroups; ++g)
#pragma unroll
          for (int jp = 0; jp < 2; ++jp) {
            uint32_t bf[4];
            const int row = ks * 16 + krow;
            const int ch = (g0 + g) * 4 + 2 * jp + (lane >> 4);
            ldmatrix_x4_trans(piece + row * 128 + ((ch ^ (row & 7)) << 4), bf);
            mma_16816_bf16(acc[g][2 * jp], vf[ks][0], vf[ks][1], vf[ks][2], vf[ks][3], bf[0], bf[1]);
            mma_16816_bf16(acc[g][2 * jp + 1], vf[ks][0], vf[ks][1], vf[ks][2], vf[ks][3], bf[2], bf[3]);
          }
    }
#pragma unroll
    for (int g = 0; g < C::kGroups; ++g) {
      const int col = n0 + wn * C::kWarpCols + g * 32 + 8 * tig;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int tok = h ? tok1 : tok0;
        float v[8] = {};
        if (tok >= 0 && col < n_hi) unpack8(ycur[g][h], v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[2 * j] += acc[g][j][2 * h];
          v[2 * j + 1] += acc[g][j][2 * h + 1];
        }
        if (gated) {
          // lanes 0, 1 of the quad hold 16 gate columns, lanes 2, 3 their up columns
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float up = __shfl_down_sync(0xffffffffu, v[e], 2, 4);
            v[e] = gated_value(v[e], up, a.act);
          }
          if (tok >= 0 && col < n_hi && tig < 2)
            *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(tok) * a.ldo + (col - 8 * tig) / 2 + 8 * tig) =
                pack8(v);
        } else if (tok >= 0 && col < n_hi) {
          if (a.act != kActNone) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = apply_act(v[e], a.act);
          }
          *reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(tok) * a.ldo + col) = pack8(v);
        }
      }
    }
    if (more) {
      if constexpr (C::kBufs == 2) {
        buf ^= 1;
      } else {
        __syncthreads();
      }
      store_p(buf);
      __syncthreads();
    }
  }
}

// ------------------------------------------------------------------ wgrad
// dP_a[r, c] = sum over a's rows of G[m, r] X[m, c].  CTA = (column tile, row
// split): the plan's rows are cut into splits of L rows whatever the adapters;
// a CTA walks its rows in stages of 64 (cp.async ring), and at each adapter's
// end adds its warps' sums in shared memory in a fixed order and writes them:
// straight to the bf16 result if the split holds all of the adapter's rows,
// else to one of the split's two f32 slots: 0 for the adapter that began in an
// earlier split, 1 for the one that goes on in a later one (there is at most
// one of each).  A reduce kernel adds an adapter's slots in order.  No atomics.
//
// Both operands have the tokens as the MMA's k: G^T and X come through
// ldmatrix.trans.  An 8-bit X (int8 codes) is read the same way as 16-bit
// pairs; each loaded word then holds the codes of two columns at two tokens,
// which byte permutes turn into the fragments of an even and an odd column
// tile: the code as a bf16 is exact ((128 + low seven bits) - (128 or 256)),
// and the row's scale of this 128-column tile multiplies G instead, in f32,
// rounded once to bf16 as the MMA's operand.
template <int R, bool I8>
struct WgradCfg {
  static constexpr int kCols = I8 ? 128 : 64;              // 128 bytes of X per row
  static constexpr int WC = (I8 && R >= 64) ? 4 : 2;       // warps along the columns
  static constexpr int WK = 8 / WC;                        // warps along the tokens
  static constexpr int kWarpCols = kCols / WC;
  static constexpr int kNT = kWarpCols / 8;
  static constexpr int kRows = 64;
  static constexpr int kStageX = kRows * 128;
  static constexpr int kStageG = kRows * R * 2;
  static constexpr int kStageS = I8 ? kRows * 4 : 0;
  static constexpr int kStage = kStageX + kStageG + kStageS;
  static constexpr int kStages = R <= 32 ? 6 : R <= 64 ? (I8 ? 4 : 5) : 3;
  static constexpr int kRedBytes = R * kCols * 4;
  static constexpr int kSmemBytes = kStages * kStage + kRedBytes;
};

struct WgradArgs {
  const void* x;
  const float* x_scales;
  const __nv_bfloat16* g;
  const int32_t* words;
  float* part;
  __nv_bfloat16* dbank;
  AdapterPlan lay;
  int64_t ldx;
  int cols, rank, A, rows_per_split;
};

template <int R>
__device__ __forceinline__ uint32_t g_swizzle(int row, int chunk) {
  constexpr int kCh = R / 8;  // 16-byte chunks per row of G
  const int f = kCh >= 8 ? (row & 7) : kCh == 4 ? ((row >> 1) & 3) : ((row >> 2) & 1);
  return static_cast<uint32_t>(row * (R * 2) + ((chunk ^ f) << 4));
}

// Four int8 codes (bytes: token 0 columns 0, 1; token 1 columns 0, 1) -> the
// bf16 pairs (token 0, token 1) of column 0 and of column 1, exact.
__device__ __forceinline__ void i8_pairs(uint32_t u, uint32_t& even, uint32_t& odd) {
  const uint32_t low = u & 0x7F7F7F7Fu, sign = u & 0x80808080u;
  const uint32_t e1 = prmt(low, 0x43u, 0x4240u), e2 = prmt(sign, 0x43u, 0x4240u);
  const uint32_t o1 = prmt(low, 0x43u, 0x4341u), o2 = prmt(sign, 0x43u, 0x4341u);
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(even) : "r"(e1), "r"(e2));
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(odd) : "r"(o1), "r"(o2));
}

__device__ __forceinline__ uint32_t scale_pair(uint32_t g, float s0, float s1) {
  return pack_bf16x2(__uint_as_float(g << 16) * s0, __uint_as_float(g & 0xFFFF0000u) * s1);
}

template <int R, bool I8>
__global__ void __launch_bounds__(256, R <= 64 ? 2 : 1) adapter_wgrad_kernel(const WgradArgs a) {
  using C = WgradCfg<R, I8>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t sbase = smem_u32(smem_raw);
  float* red = reinterpret_cast<float*>(smem_raw + C::kStages * C::kStage);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g4 = lane >> 2, tig = lane & 3;
  const int wc = warp % C::WC, wk = warp / C::WC;
  const int col0 = blockIdx.x * C::kCols;
  const int32_t* perm = a.words + a.lay.off_perm;
  const int32_t* blk = a.words + a.lay.off_blk;
  const int32_t* starts = a.words + a.lay.off_start;
  const int row_lo = blockIdx.y * a.rows_per_split;
  const int row_hi = min(row_lo + a.rows_per_split, a.words[AdapterPlan::kNoneStart]);
  grid_wait();  // G may be the output of the kernel before this one
  if (row_lo >= row_hi) return;

  // stages: 64 rows from `pos`, not past the adapter's end `end`
  struct Cursor {
    int pos, end, adapter;
  };
  auto open = [&](Cursor& c) {
    if (c.pos < row_hi) {
      c.adapter = blk[c.pos / 16];
      c.end = min(row_hi, starts[c.adapter + 1]);
    }
  };
  const int chunk = tid & 7;
  const int elem = I8 ? 1 : 2;  // bytes per element of X
  const int ncb = (a.cols + 127) / 128;
  auto load = [&](Cursor& c, int slot) {
    if (c.pos < row_hi) {
      const uint32_t sx = sbase + slot * C::kStage, sg = sx + C::kStageX, ss = sg + C::kStageG;
      const int col = col0 + chunk * (16 / elem);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = (tid >> 3) + 32 * i;
        const int token = c.pos + row < c.end ? perm[c.pos + row] : -1;
        const bool ok = token >= 0 && col < a.cols;
        const uint8_t* src = static_cast<const uint8_t*>(a.x);
        if (ok) src += (static_cast<int64_t>(token) * a.ldx + col) * elem;
        cp_async_16(sx + row * 128 + ((chunk ^ (row & 7)) << 4), src, ok);
        if constexpr (I8) {
          if (chunk == 0)
            cp_async_4z(ss + row * 4,
                        token >= 0 ? a.x_scales + static_cast<int64_t>(token) * ncb + col0 / 128 : a.x_scales,
                        token >= 0);
        }
      }
#pragma unroll
      for (int i = 0; i < (64 * (R / 8) + 255) / 256; ++i) {
        const int e = tid + 256 * i;
        const int row = e / (R / 8), ch = e % (R / 8);
        if (64 * (R / 8) % 256 != 0 && row >= 64) break;
        const int token = c.pos + row < c.end ? perm[c.pos + row] : -1;
        const bool ok = token >= 0 && ch * 8 < a.rank;
        cp_async_16(sg + g_swizzle<R>(row, ch), ok ? a.g + static_cast<int64_t>(token) * a.rank + ch * 8 : a.g, ok);
      }
      c.pos += C::kRows;
      if (c.pos >= c.end) {
        c.pos = c.end;
        open(c);
      }
    }
    cp_async_commit();
  };

  Cursor in{row_lo, 0, 0}, at{row_lo, 0, 0};
  open(in);
  open(at);
#pragma unroll
  for (int s = 0; s < C::kStages - 1; ++s) load(in, s);

  float acc[R / 16][C::kNT][4] = {};
  int step = 0;
  while (at.pos < row_hi) {
    cp_async_wait<C::kStages - 2>();
    __syncthreads();
    load(in, (step + C::kStages - 1) % C::kStages);
    const uint32_t sx = sbase + (step % C::kStages) * C::kStage, sg = sx + C::kStageX;
    const float* ss = reinterpret_cast<const float*>(smem_raw + (step % C::kStages) * C::kStage + C::kStageX + C::kStageG);
    ++step;
#pragma unroll
    for (int kb = 0; kb < C::kRows / 16 / C::WK; ++kb) {
      const int m0 = (kb * C::WK + wk) * 16;
      if (at.pos + m0 >= at.end) continue;  // warp-uniform
      uint32_t bf[C::kNT][2];
      if constexpr (!I8) {
#pragma unroll
        for (int np = 0; np < C::kNT / 2; ++np) {
          uint32_t r4[4];
          const int row = m0 + (lane & 7) + ((lane >> 3) & 1) * 8;
          const int ch = wc * (C::kWarpCols / 8) + 2 * np + (lane >> 4);
          ldmatrix_x4_trans(sx + row * 128 + ((ch ^ (row & 7)) << 4), r4);
          bf[2 * np][0] = r4[0];
          bf[2 * np][1] = r4[1];
          bf[2 * np + 1][0] = r4[2];
          bf[2 * np + 1][1] = r4[3];
        }
      } else {
        // 16-byte chunk = 16 columns = an even and an odd tile
#pragma unroll
        for (int np = 0; np < C::kNT / 4; ++np) {
          uint32_t r4[4];
          const int row = m0 + (lane & 7) + ((lane >> 3) & 1) * 8;
          const int ch = wc * (C::kWarpCols / 16) + 2 * np + (lane >> 4);
          ldmatrix_x4_trans(sx + row * 128 + ((ch ^ (row & 7)) << 4), r4);
          i8_pairs(r4[0], bf[4 * np][0], bf[4 * np + 1][0]);
          i8_pairs(r4[1], bf[4 * np][1], bf[4 * np + 1][1]);
          i8_pairs(r4[2], bf[4 * np + 2][0], bf[4 * np + 3][0]);
          i8_pairs(r4[3], bf[4 * np + 2][1], bf[4 * np + 3][1]);
        }
      }
#pragma unroll
      for (int rt = 0; rt < R / 16; ++rt) {
        // G^T: matrices (r 0-7, m 0-7), (r 8-15, m 0-7), (r 0-7, m 8-15), (r 8-15, m 8-15)
        uint32_t af[4];
        const int row = m0 + (lane & 7) + (lane >> 4) * 8;
        ldmatrix_x4_trans(sg + g_swizzle<R>(row, 2 * rt + ((lane >> 3) & 1)), af);
        if constexpr (I8) {
          const float2 s0 = *reinterpret_cast<const float2*>(ss + m0 + 2 * tig);
          const float2 s1 = *reinterpret_cast<const float2*>(ss + m0 + 8 + 2 * tig);
          af[0] = scale_pair(af[0], s0.x, s0.y);
          af[1] = scale_pair(af[1], s0.x, s0.y);
          af[2] = scale_pair(af[2], s1.x, s1.y);
          af[3] = scale_pair(af[3], s1.x, s1.y);
        }
#pragma unroll
        for (int nt = 0; nt < C::kNT; ++nt)
          mma_16816_bf16(acc[rt][nt], af[0], af[1], af[2], af[3], bf[nt][0], bf[nt][1]);
      }
    }
    at.pos += C::kRows;
    if (at.pos < at.end) continue;
    // the adapter's rows of this split are done: add the warps' sums
    const int ad = at.adapter;
#pragma unroll 1
    for (int w = 0; w < C::WK; ++w) {
      if (wk == w) {
#pragma unroll
        for (int rt = 0; rt < R / 16; ++rt)
#pragma unroll
          for (int nt = 0; nt < C::kNT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = rt * 16 + g4 + 8 * (i >> 1);
              int c;
              if constexpr (I8)  // tile pairs: even columns, odd columns of 16
                c = wc * C::kWarpCols + (nt >> 1) * 16 + 2 * (2 * tig + (i & 1)) + (nt & 1);
              else
                c = wc * C::kWarpCols + nt * 8 + 2 * tig + (i & 1);
              float* p = red + r * C::kCols + c;
              *p = (w == 0 ? 0.f : *p) + acc[rt][nt][i];
              acc[rt][nt][i] = 0.f;
            }
      }
      __syncthreads();
    }
    const bool whole = starts[ad] >= row_lo && starts[ad + 1] <= row_lo + a.rows_per_split;
    const int64_t slot = whole ? ad : 2 * static_cast<int>(blockIdx.y) + (starts[ad] < row_lo ? 0 : 1);
    const int64_t base = slot * a.rank * a.cols;
    for (int e = tid; e < R * (C::kCols / 4); e += 256) {
      const int r = e / (C::kCols / 4), c = (e % (C::kCols / 4)) * 4;
      if (r < a.rank && col0 + c < a.cols) {
        const float4 v = *reinterpret_cast<const float4*>(red + r * C::kCols + c);
        const int64_t o = base + static_cast<int64_t>(r) * a.cols + col0 + c;
        if (whole)
          *reinterpret_cast<uint2*>(a.dbank + o) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
        else
          *reinterpret_cast<float4*>(a.part + o) = v;
      }
    }
    // (the next adapter's end writes `red` again only after the barrier at the
    // top of the loop, which every thread reaches after its reads here)
    at.pos = at.end;
    open(at);
  }
  cp_async_wait<0>();
}

// Adds the slots of adapters that several splits share, in split order; zeros
// for adapters without rows.  blockIdx.y: adapter.
__global__ void __launch_bounds__(256)
    adapter_wgrad_reduce_kernel(const int32_t* __restrict__ words, AdapterPlan lay, int rows_per_split,
                                const float* __restrict__ part, __nv_bfloat16* __restrict__ dbank,
                                int64_t elems) {
  const int ad = blockIdx.y;
  const int lo = words[lay.off_start + ad], hi = words[lay.off_start + ad + 1];
  grid_wait();
  const int s0 = lo / rows_per_split, s1 = hi > lo ? (hi - 1) / rows_per_split : s0;
  if (hi > lo && s0 == s1) return;
  for (int64_t i = (blockIdx.x * 256ll + threadIdx.x) * 4; i < elems; i += gridDim.x * 1024ll) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (hi > lo)
      for (int s = s0; s <= s1; ++s) {
        const float4 u = __ldcg(reinterpret_cast<const float4*>(part + static_cast<int64_t>(2 * s + (s == s0 ? 1 : 0)) * elems + i));
        v.x += u.x;
        v.y += u.y;
        v.z += u.z;
        v.w += u.w;
      }
    *reinterpret_cast<uint2*>(dbank + static_cast<int64_t>(ad) * elems + i) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
}

}  // namespace dq
