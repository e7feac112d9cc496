// dq_adapter.cu -- host side of include/dq_adapter.h: argument validation,
// launch planning and launches of the adapter and activation-checkpoint kernels
// (the input gradients are in dq_dgrad.cu).
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <mutex>

#include "../../include/dq_adapter.h"
#include "dq_adapter.cuh"
#include "dq_checkpoint.cuh"
#include "dq_internal.h"
#include "dq_launch.h"

namespace dq {
namespace {

constexpr int64_t kMaxTokens = 1 << 30;
constexpr int64_t kMaxRequests = 1 << 20;
constexpr int kMaxAdapters = 65535;
constexpr int kMaxRank = 128;
constexpr int kMaxCluster = 8;

int plan_shape(int64_t M, int64_t R, int A) {
  return M < 0 || M > kMaxTokens || R < 0 || R > kMaxRequests || A < 1 || A > kMaxAdapters ? DQ_ERR_SHAPE : DQ_OK;
}
int bank_shape(int64_t M, int64_t R, int64_t K, int64_t N, int r, int A) {
  if (plan_shape(M, R, A) != DQ_OK || K <= 0 || N <= 0 || K % 8 != 0 || N % 8 != 0 || r <= 0 || r % 8 != 0 ||
      r > kMaxRank || K > INT32_MAX || N > INT32_MAX)
    return DQ_ERR_SHAPE;
  return DQ_OK;
}
bool row_stride_ok(int64_t ld, int64_t width) { return ld >= width && ld % 8 == 0; }

// Rank the kernels are instantiated for: the next of 16, 32, 64, 128 (columns
// past the rank are zeros).
int rank_class(int r) { return r <= 16 ? 16 : r <= 32 ? 32 : r <= 64 ? 64 : 128; }

// 128-row tiles where the groups fill at least half of one on average, else
// 16-row tiles.
bool large_tiles(int64_t M, int64_t R, int A) {
  return M >= 64 * std::max<int64_t>(1, std::min<int64_t>(A, R));
}

// Feature splits of the large-tile down kernel, the CTAs of a cluster: the size
// with the least waves x (stages of 64 features per CTA + a fixed cost of
// eight), each split at least 256 features deep.  How many clusters are
// resident at once decides, because a cluster stays within a graphics
// processing cluster of the device: at 4608 tokens 36 clusters of eight run in
// two waves, of six in one.  clusters[c]: how many of c CTAs fit.
struct DownPlan {
  int tiles, splits, k_per_split;
};
DownPlan down_plan(int64_t M, int64_t R, int A, int64_t F, const int* clusters) {
  DownPlan p;
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>(A, R));
  const int64_t likely = ceil_div(M, kTileRows) + groups / 2;
  p.tiles = static_cast<int>(adapter_plan_layout(M, R, A).max_tiles);
  int64_t best = INT64_MAX, s = 1;
  for (int64_t c : {1, 2, 4, 6, 8}) {
    if (c > std::max<int64_t>(1, F / 256)) break;
    const int64_t cost = ceil_div(likely, std::max(1, clusters[c])) * (ceil_div(ceil_div(F, c), 64) + 8);
    if (cost < best) {
      best = cost;
      s = c;
    }
  }
  p.k_per_split = static_cast<int>(ceil_div(ceil_div(F, s), 64) * 64);
  p.splits = static_cast<int>(ceil_div(F, p.k_per_split));
  return p;
}

// Row splits of the weight-gradient kernel: the count (up to 16) that leaves
// the smallest share of the resident CTA slots idle in its last wave, for
// splits of at least 256 rows.  col_tiles: of all problems of the launch.
struct WgradPlan {
  int splits, rows_per_split;
};
WgradPlan wgrad_plan(int64_t M, int64_t R, int A, int64_t col_tiles, int rc, bool i8, int sms) {
  const AdapterPlan lay = adapter_plan_layout(M, R, A);
  const int slots = sms * (rc <= 64 || !i8 ? 2 : 1);  // WgradCfg::kMinCtas
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(16, M / 256));
  double best = 0;
  int splits = 1;
  for (int64_t s = 1; s <= most; ++s) {
    const int64_t ctas = col_tiles * s;
    const double fill = static_cast<double>(ctas) / static_cast<double>(ceil_div(ctas, slots) * slots);
    if (fill > best + 0.02) {
      best = fill;
      splits = static_cast<int>(s);
    }
  }
  WgradPlan p;
  p.rows_per_split = static_cast<int>(ceil_div(ceil_div(lay.cap, splits), 64) * 64);
  p.splits = static_cast<int>(ceil_div(lay.cap, p.rows_per_split));
  return p;
}
int64_t col_tiles(int64_t cols) { return ceil_div(cols, 128); }

// Resident clusters of the down kernel by their (even) size, once per device.
// The runtime's occupancy query counts one CTA per SM for a kernel that
// allocates tensor memory, though two fit by its shared memory and run, so the
// count for c CTAs is the one it gives for c / 2.
template <int R>
int down_clusters(const int** out) {
  using C = DownCfg<R>;
  static std::atomic<int> set[kMaxDevices], probed[kMaxDevices];
  static int table[kMaxDevices][kMaxCluster + 1];
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return DQ_ERR_CUDA;
  const int rc = allow_smem(adapter_down_kernel<R>, C::kSmemBytes, set);
  if (rc != DQ_OK) return rc;
  if (!probed[dev].load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lk(mu);
    for (int half = 1; half <= kMaxCluster / 2; ++half) {
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 1;
      attr[0].val.clusterDim.y = half;
      attr[0].val.clusterDim.z = 1;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1024, half);
      cfg.blockDim = dim3(C::kThreads);
      cfg.dynamicSmemBytes = C::kSmemBytes;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, adapter_down_kernel<R>, &cfg) != cudaSuccess) return DQ_ERR_LAUNCH;
      table[dev][2 * half] = n;
      if (half == 1) table[dev][1] = 2 * n;
    }
    probed[dev].store(1, std::memory_order_release);
  }
  *out = table[dev];
  return DQ_OK;
}

template <int R>
int launch_down(DownArgs a, int64_t M, int64_t requests, cudaStream_t st) {
  using C = DownCfg<R>;
  const int* clusters = nullptr;
  const int rc = down_clusters<R>(&clusters);
  if (rc != DQ_OK) return rc;
  const DownPlan p = down_plan(M, requests, a.A, a.K, clusters);
  a.k_per_split = p.k_per_split;
  return launch(adapter_down_kernel<R>, dim3(p.tiles, p.splits), C::kThreads, C::kSmemBytes, st, false,
                dim3(1, p.splits), a);
}

template <int R>
int launch_up(UpArgs a, int tiles, int64_t M, int64_t requests, int sms, cudaStream_t st) {
  using C = UpCfg<R>;
  static std::atomic<int> set[kMaxDevices];
  const int rc = allow_smem(adapter_up_kernel<R>, C::kSmemBytes, set);
  if (rc != DQ_OK) return rc;
  // 64-column steps per CTA: the fewest that put the whole launch into one wave
  // if eight are enough (4608 x 4096 at r = 64: six steps 22 us, four, a wave
  // and a third, 25), else six (4613 x 16384 at r = 32, with / without GELU, down
  // product included: six 77 / 67 us, four, whose CTAs' first loads weigh more,
  // 80 / 69, sixteen, which leave the last wave emptier, 82 / 74)
  const int64_t total = ceil_div(a.N, C::kStepCols), slots = static_cast<int64_t>(sms) * C::kMinCtas;
  const int64_t most = ceil_div(M, kTileRows) + std::min<int64_t>(a.A, requests) + 1;
  int64_t steps = 1;
  while (steps <= 8 && most * ceil_div(total, steps) > slots) ++steps;
  if (steps > 8) steps = 6;
  a.cols_per_cta = static_cast<int>(steps * C::kStepCols);
  return launch(adapter_up_kernel<R>, dim3(tiles, static_cast<unsigned>(ceil_div(total, steps))), 256, C::kSmemBytes, st,
                true, dim3(1), a);
}

// Resident clusters of the small-batch kernel, once per device (it allocates no
// tensor memory, so the runtime's count holds).
template <int R>
int small_clusters(int* out) {
  using C = SmallCfg<R>;
  static std::atomic<int> set[kMaxDevices], count[kMaxDevices];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return DQ_ERR_CUDA;
  const int rc = allow_smem(adapter_small_kernel<R>, C::kSmemBytes, set);
  if (rc != DQ_OK) return rc;
  int n = count[dev].load(std::memory_order_acquire);
  if (n == 0) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kSmallCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1024 * kSmallCluster);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, adapter_small_kernel<R>, &cfg) != cudaSuccess || n < 1) return DQ_ERR_LAUNCH;
    count[dev].store(n, std::memory_order_release);
  }
  *out = n;
  return DQ_OK;
}

template <int R>
int launch_small(SmallArgs a, int64_t M, int64_t R_, cudaStream_t st) {
  using C = SmallCfg<R>;
  int resident = 0;
  const int rc = small_clusters<R>(&resident);
  if (rc != DQ_OK) return rc;
  a.k_per_rank = static_cast<int>(ceil_div(ceil_div(a.K, kSmallCluster), 32) * 32);
  // clusters per tile: more than one (each repeats the down projection) only
  // while the CTAs have more than one step of columns and all are resident at
  // once (rank 64, N = 12288, one token for each of 4 adapters 9.2 us, in two
  // waves 18.7; of 8 adapters 12.5 and 21.9; N = 4096 8.0 and 12.7)
  const int64_t tiles = std::max<int64_t>(ceil_div(M, kBlockRows), std::min<int64_t>(std::min<int64_t>(a.A, R_), M));
  int clusters = 1;
  while (clusters < 8 && a.N > clusters * kSmallCluster * C::kStepCols && 2 * clusters * tiles <= resident) clusters *= 2;
  a.cols_per_cta = static_cast<int>(ceil_div(ceil_div(a.N, clusters * kSmallCluster), 64) * 64);
  a.ctas_per_tile = clusters * kSmallCluster;
  const dim3 grid(static_cast<unsigned>(a.lay.cap / kBlockRows) * a.ctas_per_tile);
  return launch(adapter_small_kernel<R>, grid, 256, C::kSmemBytes, st, false, dim3(kSmallCluster), a);
}

template <int R, bool I8>
int launch_wgrad(const WgradArgs& a, int splits, cudaStream_t st) {
  using C = WgradCfg<R, I8>;
  static std::atomic<int> set[kMaxDevices];
  const int rc = allow_smem(adapter_wgrad_kernel<R, I8>, C::kSmemBytes, set);
  if (rc != DQ_OK) return rc;
  return launch(adapter_wgrad_kernel<R, I8>, dim3(a.first.col_tiles + a.second.col_tiles, splits), C::kThreads,
                C::kSmemBytes, st, true, dim3(1), a);
}

// Calls f.template operator()<R>() for the rank class.
template <typename F>
int by_rank(int r, F&& f) {
  switch (rank_class(r)) {
    case 16: return f(std::integral_constant<int, 16>());
    case 32: return f(std::integral_constant<int, 32>());
    case 64: return f(std::integral_constant<int, 64>());
  }
  return f(std::integral_constant<int, 128>());
}

// Workspace of the backward pass: g [M, r] in bf16 and in f32, and one region
// for each weight gradient's partial sums.
struct BackwardWs {
  WgradPlan up, down;  // splits of dup and of ddown
  size_t g, g32, up_bytes, down_bytes, total;
};
BackwardWs backward_ws(int64_t M, int64_t R, int64_t K, int64_t N, int r, int A, bool i8, int sms) {
  BackwardWs w;
  const int rc = rank_class(r);
  if (i8) {  // a launch each
    w.up = wgrad_plan(M, R, A, col_tiles(N), rc, false, sms);
    w.down = wgrad_plan(M, R, A, col_tiles(K), rc, true, sms);
  } else {  // one launch
    w.up = w.down = wgrad_plan(M, R, A, col_tiles(N) + col_tiles(K), rc, false, sms);
  }
  auto part = [&](const WgradPlan& p, int64_t cols) { return up256(static_cast<size_t>(2) * p.splits * r * cols * 4); };
  w.g = up256(static_cast<size_t>(M) * r * 2);
  w.g32 = i8 ? up256(static_cast<size_t>(M) * r * 4) : 0;
  w.up_bytes = part(w.up, N);
  w.down_bytes = part(w.down, K);
  w.total = w.g + w.g32 + w.up_bytes + w.down_bytes;
  return w;
}

// hidden = scale x . P^T (down), out = act(y + hidden . Q) (up), on one plan;
// without an out the first alone.
// hidden: where the low-rank intermediate goes, complete (zero rows without an
// adapter) if want_hidden; the small-batch kernel takes NULL.  between: launches
// that read x again, put right behind the large-tile down kernel while x is
// still in L2 (behind everything for small batches).
template <typename Between>
int down_up(const void* x, int64_t ldx, int64_t F_in, const void* P, const void* y, int64_t ldy, int64_t F_out,
            const void* Q, const float* scale, int64_t M, int64_t R, int r, int A, const int32_t* words, int act,
            void* out, int64_t ldo, void* hidden, bool want_hidden, float* hidden32, int sms, cudaStream_t st,
            Between between) {
  const AdapterPlan lay = adapter_plan_layout(M, R, A);
  const int with_none = out != nullptr && (act != kActNone || out != y || want_hidden);
  if (!large_tiles(M, R, A)) {
    SmallArgs a = {};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.y = static_cast<const __nv_bfloat16*>(y);
    a.down = static_cast<const __nv_bfloat16*>(P);
    a.up = static_cast<const __nv_bfloat16*>(Q);
    a.scale = scale;
    a.words = words;
    a.out = static_cast<__nv_bfloat16*>(out);
    a.hidden = want_hidden ? static_cast<__nv_bfloat16*>(hidden) : nullptr;
    a.hidden32 = hidden32;
    a.lay = lay;
    a.ldx = ldx;
    a.ldy = ldy;
    a.ldo = ldo;
    a.K = static_cast<int>(F_in);
    a.N = out == nullptr ? 0 : static_cast<int>(F_out);  // (no columns: the hidden tile is all)
    a.rank = r;
    a.A = A;
    a.act = act;
    a.with_none = with_none;
    const int e = by_rank(r, [&](auto rc) { return launch_small<decltype(rc)::value>(a, M, R, st); });
    return e != DQ_OK ? e : between();
  }
  DownArgs d = {};
  int e = error_word(&d.error);
  if (e != DQ_OK) return e;
  d.x = static_cast<const __nv_bfloat16*>(x);
  d.bank = static_cast<const __nv_bfloat16*>(P);
  d.scale = scale;
  d.words = words;
  d.hidden = static_cast<__nv_bfloat16*>(hidden);
  d.hidden32 = hidden32;
  d.lay = lay;
  d.ldx = ldx;
  d.K = static_cast<int>(F_in);
  d.rank = r;
  d.A = A;
  UpArgs u = {};
  u.y = static_cast<const __nv_bfloat16*>(y);
  u.bank = static_cast<const __nv_bfloat16*>(Q);
  u.hidden = d.hidden;
  u.words = words;
  u.out = static_cast<__nv_bfloat16*>(out);
  u.zero_hidden = want_hidden ? d.hidden : nullptr;
  u.lay = lay;
  u.ldy = ldy;
  u.ldo = ldo;
  u.N = static_cast<int>(F_out);
  u.rank = r;
  u.A = A;
  u.act = act;
  u.with_none = with_none;
  return by_rank(r, [&](auto rc) {
    constexpr int R_ = decltype(rc)::value;
    int e2 = launch_down<R_>(d, M, R, st);
    if (e2 == DQ_OK) e2 = between();
    return e2 != DQ_OK || out == nullptr ? e2 : launch_up<R_>(u, static_cast<int>(lay.max_tiles), M, R, sms, st);
  });
}

}  // namespace
}  // namespace dq

using namespace dq;

extern "C" {

size_t dq_adapter_plan_bytes(int64_t M, int64_t R, int A) {
  if (plan_shape(M, R, A) != DQ_OK) return 0;
  return static_cast<size_t>(adapter_plan_layout(M, R, A).words) * 4;
}

int dq_adapter_plan(const int32_t* ids, const int32_t* offsets, int64_t R, int64_t M, int A, void* plan,
                    size_t plan_bytes, dq_stream_t stream) {
  int rc = plan_shape(M, R, A);
  if (rc != DQ_OK) return rc;
  if (offsets == nullptr || plan == nullptr || (R > 0 && ids == nullptr)) return DQ_ERR_ARG;
  if (!aligned(ids, 4) || !aligned(offsets, 4) || !aligned(plan, 16)) return DQ_ERR_ALIGN;
  if (plan_bytes < dq_adapter_plan_bytes(M, R, A)) return DQ_ERR_WORKSPACE;
  int sms = 0;
  if ((rc = device_sms(&sms)) != DQ_OK) return rc;
  unsigned int* error = nullptr;
  if ((rc = error_word(&error)) != DQ_OK) return rc;
  const AdapterPlan lay = adapter_plan_layout(M, R, A);
  int32_t* words = static_cast<int32_t*>(plan);
  const int grid = static_cast<int>(ceil_div(A + 1, 8));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  adapter_count_kernel<<<grid, 256, 0, st>>>(ids, offsets, static_cast<int>(R), static_cast<int>(M), A,
                                             words + lay.off_counts, error);
  adapter_place_kernel<<<grid, 256, 0, st>>>(ids, offsets, static_cast<int>(R), static_cast<int>(M), A, words,
                                             lay, error);
  return cudaGetLastError() == cudaSuccess ? DQ_OK : DQ_ERR_LAUNCH;
}

size_t dq_adapter_add_workspace(int64_t M, int64_t R, int r, int A) {
  if (plan_shape(M, R, A) != DQ_OK || r <= 0 || r > kMaxRank || !large_tiles(M, R, A)) return 0;
  return static_cast<size_t>(M) * r * 2;
}

int dq_adapter_add(const void* y, int64_t ldy, const void* x, int64_t ldx, int64_t M, int64_t R, int64_t K,
                   int64_t N, const void* down, const void* up, const float* scale, int r, int A,
                   const void* plan, int act, void* out, int64_t ldo, void* hidden, void* workspace,
                   size_t workspace_bytes, dq_stream_t stream) {
  if (act < kActNone || act > kActGeGluTanh) return DQ_ERR_ARG;
  int rc = bank_shape(M, R, K, N, r, A);
  if (rc != DQ_OK) return rc;
  const bool gated = act_is_gated(act);
  if (gated && N % 32 != 0) return DQ_ERR_SHAPE;
  if (!row_stride_ok(ldy, N) || !row_stride_ok(ldx, K) || !row_stride_ok(ldo, gated ? N / 2 : N)) return DQ_ERR_SHAPE;
  if (M == 0) return DQ_OK;
  if (y == nullptr || x == nullptr || down == nullptr || up == nullptr || scale == nullptr || plan == nullptr ||
      out == nullptr)
    return DQ_ERR_ARG;
  if (gated && out == y) return DQ_ERR_ARG;  // rows change their width
  if (out == y && ldo != ldy) return DQ_ERR_SHAPE;
  if (!aligned(y, 16) || !aligned(x, 16) || !aligned(down, 16) || !aligned(up, 16) || !aligned(scale, 4) ||
      !aligned(plan, 16) || !aligned(out, 16) || !aligned(hidden, 16))
    return DQ_ERR_ALIGN;
  int sms = 0;
  if ((rc = device_sms(&sms)) != DQ_OK) return rc;
  const size_t need = hidden == nullptr ? dq_adapter_add_workspace(M, R, r, A) : 0;
  if (need > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < need)) return DQ_ERR_WORKSPACE;
  return down_up(x, ldx, K, down, y, ldy, N, up, scale, M, R, r, A, static_cast<const int32_t*>(plan), act, out,
                 ldo, hidden != nullptr ? hidden : workspace, hidden != nullptr, nullptr, sms,
                 static_cast<cudaStream_t>(stream), [] { return static_cast<int>(DQ_OK); });
}

size_t dq_adapter_backward_workspace(int64_t M, int64_t R, int64_t K, int64_t N, int r, int A) {
  int sms = 0;
  if (bank_shape(M, R, K, N, r, A) != DQ_OK || device_sms(&sms) != DQ_OK) return 0;
  return std::max(backward_ws(M, R, K, N, r, A, false, sms).total, backward_ws(M, R, K, N, r, A, true, sms).total);
}

int dq_adapter_backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const float* x_scales,
                        const void* hidden, int64_t M, int64_t R, int64_t K, int64_t N, const void* down,
                        const void* up, const float* scale, int r, int A, const void* plan, const void* dx,
                        int64_t lddx, void* dx_out, int64_t lddxo, void* ddown, void* dup, void* workspace,
                        size_t workspace_bytes, dq_stream_t stream) {
  int rc = bank_shape(M, R, K, N, r, A);
  if (rc != DQ_OK) return rc;
  const bool i8 = x_scales != nullptr;
  const bool want_w = ddown != nullptr, want_x = dx != nullptr || dx_out != nullptr;
  if (!row_stride_ok(lddy, N) || (i8 && (K % 16 != 0 || ldx < K || ldx % 16 != 0)) ||
      (want_w && !i8 && !row_stride_ok(ldx, K)))
    return DQ_ERR_SHAPE;
  if (want_x && (!row_stride_ok(lddx, K) || !row_stride_ok(lddxo, K))) return DQ_ERR_SHAPE;
  if ((ddown == nullptr) != (dup == nullptr) || (M > 0 && !want_x && !want_w)) return DQ_ERR_ARG;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    if (want_w && (cudaMemsetAsync(ddown, 0, static_cast<size_t>(A) * r * K * 2, st) != cudaSuccess ||
                   cudaMemsetAsync(dup, 0, static_cast<size_t>(A) * r * N * 2, st) != cudaSuccess))
      return DQ_ERR_CUDA;
    return DQ_OK;
  }
  if (dy == nullptr || down == nullptr || up == nullptr || scale == nullptr || plan == nullptr ||
      (want_x && (dx == nullptr || dx_out == nullptr)) || (want_w && (x == nullptr || hidden == nullptr)))
    return DQ_ERR_ARG;
  if (want_x && dx == dx_out && lddx != lddxo) return DQ_ERR_SHAPE;
  if (!aligned(dy, 16) || !aligned(x, 16) || !aligned(x_scales, 4) || !aligned(hidden, 16) || !aligned(down, 16) ||
      !aligned(up, 16) || !aligned(scale, 4) || !aligned(plan, 16) || !aligned(dx, 16) || !aligned(dx_out, 16) ||
      !aligned(ddown, 16) || !aligned(dup, 16))
    return DQ_ERR_ALIGN;
  int sms = 0;
  if ((rc = device_sms(&sms)) != DQ_OK) return rc;
  const BackwardWs w = backward_ws(M, R, K, N, r, A, i8, sms);
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < w.total) return DQ_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int32_t* words = static_cast<const int32_t*>(plan);
  float* g32 = i8 ? reinterpret_cast<float*>(ws + w.g) : nullptr;
  WgradArgs a = {};
  if ((rc = error_word(&a.error)) != DQ_OK) return rc;
  a.words = words;
  a.lay = adapter_plan_layout(M, R, A);
  a.rank = r;
  a.A = A;
  // one split holds every adapter's rows: what is left to the reduce kernel are
  // zeros, which the CTAs write themselves while those are few (512 rows of
  // zeros, 128 KB a CTA; a launch less: 24 -> 20 us for 48 tokens from Python)
  a.alone = w.up.splits == 1 && w.down.splits == 1 && static_cast<int64_t>(A) * r <= 512;
  WgradProblem pu = {}, pd = {};
  pu.x = dy;
  pu.ldx = lddy;
  pu.g = static_cast<const __nv_bfloat16*>(hidden);
  pu.part = reinterpret_cast<float*>(ws + w.g + w.g32);
  pu.dbank = static_cast<__nv_bfloat16*>(dup);
  pu.cols = static_cast<int>(N);
  pu.col_tiles = static_cast<int>(col_tiles(N));
  pu.rows_per_split = w.up.rows_per_split;
  pd.x = x;
  pd.ldx = ldx;
  pd.x_scales = x_scales;
  pd.g = reinterpret_cast<const __nv_bfloat16*>(ws);
  pd.g32 = g32;
  pd.part = reinterpret_cast<float*>(ws + w.g + w.g32 + w.up_bytes);
  pd.dbank = static_cast<__nv_bfloat16*>(ddown);
  pd.cols = static_cast<int>(K);
  pd.col_tiles = static_cast<int>(col_tiles(K));
  pd.rows_per_split = w.down.rows_per_split;
  // dup needs hidden and dy alone: it follows the product that has just read dy
  // (an 8-bit x takes its own kernel; with a bf16 x one launch computes both)
  a.first = pu;
  auto first = [&] {
    if (!want_w || !i8) return static_cast<int>(DQ_OK);
    return by_rank(r, [&](auto rank) { return launch_wgrad<decltype(rank)::value, false>(a, w.up.splits, st); });
  };
  rc = down_up(dy, lddy, N, up, dx, lddx, K, down, scale, M, R, r, A, words, kActNone, dx_out, lddxo, ws, want_w,
               want_w ? g32 : nullptr, sms, st, first);
  if (rc != DQ_OK || !want_w) return rc;
  rc = by_rank(r, [&](auto rank) {
    constexpr int R_ = decltype(rank)::value;
    if (i8) {
      a.first = pd;
      return launch_wgrad<R_, true>(a, w.down.splits, st);
    }
    a.second = pd;
    return launch_wgrad<R_, false>(a, w.up.splits, st);
  });
  if (rc != DQ_OK || a.alone) return rc;
  a.first = pu;
  a.second = pd;
  const int64_t elems = static_cast<int64_t>(r) * std::max(K, N);
  const unsigned bx = static_cast<unsigned>(std::min<int64_t>(ceil_div(elems, 1024), 512));
  return launch(adapter_wgrad_reduce_kernel, dim3(bx, A, 2), 256, 0, st, true, dim3(1), a);
}

int dq_checkpoint_pack(const void* x, int64_t ldx, int64_t M, int64_t K, int8_t* codes, float* scales,
                       dq_stream_t stream) {
  if (M < 0 || M > INT32_MAX || K <= 0 || K > INT32_MAX || K % 16 != 0 || !row_stride_ok(ldx, K)) return DQ_ERR_SHAPE;
  if (M == 0) return DQ_OK;
  if (x == nullptr || codes == nullptr || scales == nullptr) return DQ_ERR_ARG;
  if (!aligned(x, 16) || !aligned(codes, 16) || !aligned(scales, 4)) return DQ_ERR_ALIGN;
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc != DQ_OK) return rc;
  const int nrun = static_cast<int>(ceil_div(K, kCkptRun));
  const int64_t runs = M * nrun;
  const int grid = static_cast<int>(std::min<int64_t>(ceil_div(runs, 32), static_cast<int64_t>(sms) * 6));  // resident CTAs
  checkpoint_pack_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      static_cast<const __nv_bfloat16*>(x), ldx, M, nrun, static_cast<int>(K), aligned(x, 32) && ldx % 16 == 0, codes,
      scales);
  return cudaGetLastError() == cudaSuccess ? DQ_OK : DQ_ERR_LAUNCH;
}

int dq_checkpoint_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K, void* out, int64_t ldo,
                         dq_stream_t stream) {
  if (M < 0 || M > INT32_MAX || K <= 0 || K > INT32_MAX || K % 16 != 0 || !row_stride_ok(ldo, K)) return DQ_ERR_SHAPE;
  if (M == 0) return DQ_OK;
  if (codes == nullptr || scales == nullptr || out == nullptr) return DQ_ERR_ARG;
  if (!aligned(codes, 16) || !aligned(scales, 4) || !aligned(out, 16)) return DQ_ERR_ALIGN;
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc != DQ_OK) return rc;
  const int64_t total = M * (K / 16);
  const int grid = static_cast<int>(std::min<int64_t>(ceil_div(total, 256), static_cast<int64_t>(sms) * 4));  // resident CTAs
  checkpoint_unpack_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(
      codes, scales, M, static_cast<int>(K), static_cast<int>(ceil_div(K, kCkptRun)),
      aligned(out, 32) && ldo % 16 == 0, static_cast<__nv_bfloat16*>(out), ldo);
  return cudaGetLastError() == cudaSuccess ? DQ_OK : DQ_ERR_LAUNCH;
}

}  // extern "C"
