// dq_dgrad.cu -- host side of the quantized linears' input gradients
// (include/dq_adapter.h): argument validation, planning and launches.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "../../include/dq_adapter.h"
#include "dq_dgrad.cuh"
#include "dq_internal.h"
#include "dq_launch.h"

namespace dq {
namespace {

constexpr int kFusedTokens = 512;  // tokens per CTA: the columns of tensor memory

// Whether decode and product go in one launch.  Two launches (NF4, us against
// the fused one): 333 x 4096 x 4096 28 / 20, 512 tokens 28 / 28; 512 x 16384 x
// 4096 97 / 71, x 1024 x 2048 12 / 17 (the sums' way out does not shrink with
// N), 256 x 1024 x 2048 12 / 11; 1024 x 4096 x 4096, decoded twice, 37 / 38.
bool fused_wins(int64_t M, int64_t N) {
  return N <= (1 << 30) && (M <= 256 || (M <= kFusedTokens && N >= 2048));  // (rows are counted in 32 bits)
}

// Tokens per CTA (all of them), ring stages and CTAs of a cluster along N: the
// size with the least waves x (steps of 64 n per CTA + a fixed cost of eight).
// A cluster stays within a graphics processing cluster of the device, so of the
// larger ones not all SMs find a place (32 clusters of four run in one wave,
// sixteen of eight in two).
struct FusedPlan {
  int tok_n, n_mma, feature_tiles, stages, stage_bytes, splits, per_split, red_tokens;
  uint32_t tmem_cols;
  size_t smem;
};
FusedPlan fused_plan(int fmt, int64_t M, int64_t N, int64_t K, int sms) {
  FusedPlan p = {};
  p.n_mma = M <= 256 ? 1 : 2;
  p.tok_n = static_cast<int>(ceil_div(ceil_div(M, p.n_mma), 16) * 16);
  const int tokens = p.tok_n * p.n_mma;
  p.feature_tiles = static_cast<int>(ceil_div(K, kDgradFeatures));
  p.stage_bytes = kDgradWBytes + tokens * 128;
  const int behind = kDgradLutAt + (fmt == kFmtNF4 ? kNf4LutBytes : 0), room = 226 * 1024 - behind;
  p.stages = std::min(kDgradMaxStages, room / p.stage_bytes);  // 2 (512 tokens) or more
  static_assert(2 * (kDgradWBytes + kFusedTokens * 128) <= 226 * 1024 - kDgradLutAt - kNf4LutBytes &&
                kDgradGroups <= 2, "a stage per group of decoding warps");
  p.smem = static_cast<size_t>(p.stages) * p.stage_bytes + behind + 1024;
  p.red_tokens = std::min(tokens, p.stages * p.stage_bytes / (kDgradFeatures * 4) / 16 * 16);
  p.tmem_cols = 32;
  while (static_cast<int>(p.tmem_cols) < tokens) p.tmem_cols *= 2;
  const int64_t blocks = ceil_div(N, kDgradRows);
  int64_t best = INT64_MAX;
  for (int c = 1; c <= 8; c *= 2) {
    const int64_t per = ceil_div(blocks, c);
    if ((c - 1) * per >= blocks) break;  // a rank without work
    const int64_t slots = static_cast<int64_t>(sms) * (c > 4 ? 15 : c > 2 ? 18 : 20) / 20;
    const int64_t cost = ceil_div(p.feature_tiles * c, slots) * (per + 8);
    if (cost < best) {
      best = cost;
      p.splits = c;
      p.per_split = static_cast<int>(per);
    }
  }
  return p;
}

template <int FMT>
int launch_fused(const FusedPlan& p, const void* dy, int64_t M, int64_t N, const uint8_t* w, const void* absmax,
                 int sbf, float scale, int64_t K, void* dx, cudaStream_t st) {
  static std::atomic<int> set[kMaxDevices];
  int rc = allow_smem(dgrad_fused_kernel<FMT>, 227 * 1024, set);
  if (rc != DQ_OK) return rc;
  DgradArgs a = {};
  if ((rc = error_word(&a.error)) != DQ_OK) return rc;
  CUtensorMap map;
  if (!bf16_tile_map(&map, dy, N, M, N * 2, p.tok_n)) return DQ_ERR_CUDA;
  a.w = w;
  a.absmax = absmax;
  a.dx = static_cast<__nv_bfloat16*>(dx);
  a.fp8_scale = scale;
  a.scale_bf16 = sbf;
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.tok_n = p.tok_n;
  a.n_mma = p.n_mma;
  a.stages = p.stages;
  a.stage_bytes = p.stage_bytes;
  a.per_split = p.per_split;
  a.red_tokens = p.red_tokens;
  a.tmem_cols = p.tmem_cols;
  return launch(dgrad_fused_kernel<FMT>, dim3(p.feature_tiles, p.splits), kDgradThreads, p.smem, st,
                false, dim3(1, p.splits), map, a);
}

int dgrad_impl(int fmt, const void* dy, int64_t M, int64_t N, const uint8_t* w, const void* absmax, int sbf,
                      float scale, int64_t K, void* dx, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  if (M < 0 || N <= 0 || K <= 0 || N % 8 != 0 || K % (fmt == kFmtNF4 ? 64 : 16) != 0 || M > INT32_MAX ||
      N > INT32_MAX || K > INT32_MAX || ceil_div(N, 128) > 65535)
    return DQ_ERR_SHAPE;
  if (M == 0) return DQ_OK;
  if (dy == nullptr || w == nullptr || dx == nullptr || (fmt == kFmtNF4 && absmax == nullptr)) return DQ_ERR_ARG;
  if (!aligned(dy, 16) || !aligned(w, 16) || !aligned(dx, 16) || !aligned(absmax, sbf ? 2 : 4)) return DQ_ERR_ALIGN;
  int sms = 0;
  const int rc = device_sms(&sms);
  if (rc != DQ_OK) return rc;
  if (fused_wins(M, N)) {
    const FusedPlan p = fused_plan(fmt, M, N, K, sms);
    return fmt == kFmtNF4 ? launch_fused<kFmtNF4>(p, dy, M, N, w, absmax, sbf, scale, K, dx, st)
                          : launch_fused<kFmtFP8>(p, dy, M, N, w, absmax, sbf, scale, K, dx, st);
  }
  if (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < dq_linear_dgrad_workspace(N, K))
    return DQ_ERR_WORKSPACE;
  const dim3 grid(static_cast<unsigned>(ceil_div(K, 64)), static_cast<unsigned>(ceil_div(N, 128)));
  if (fmt == kFmtNF4)
    decode_transposed_kernel<kFmtNF4><<<grid, 256, 0, st>>>(w, absmax, sbf, 0.f, static_cast<int>(N),
                                                            static_cast<int>(K),
                                                            static_cast<__nv_bfloat16*>(workspace));
  else
    decode_transposed_kernel<kFmtFP8><<<grid, 256, 0, st>>>(w, nullptr, 0, scale, static_cast<int>(N),
                                                            static_cast<int>(K),
                                                            static_cast<__nv_bfloat16*>(workspace));
  if (cudaGetLastError() != cudaSuccess) return DQ_ERR_LAUNCH;
  return bf16_gemm(dy, M, N, workspace, K, dx, K, st);
}

}  // namespace
}  // namespace dq

using namespace dq;

extern "C" {

size_t dq_linear_dgrad_workspace(int64_t N, int64_t K) {
  return N <= 0 || K <= 0 ? 0 : up256(static_cast<size_t>(N) * K * 2);
}

size_t dq_linear_dgrad_workspace_for(int64_t M, int64_t N, int64_t K) {
  return M <= 0 || fused_wins(M, N) ? 0 : dq_linear_dgrad_workspace(N, K);
}

int dq_linear_nf4_dgrad(const void* dy, int64_t M, int64_t N, const uint8_t* packed, const void* absmax,
                        int scale_dtype, int64_t K, void* dx, void* workspace, size_t workspace_bytes,
                        dq_stream_t stream) {
  if (scale_dtype != DQ_DTYPE_F32 && scale_dtype != DQ_DTYPE_BF16) return DQ_ERR_ARG;
  return dgrad_impl(kFmtNF4, dy, M, N, packed, absmax, scale_dtype == DQ_DTYPE_BF16, 0.f, K, dx, workspace,
                    workspace_bytes, static_cast<cudaStream_t>(stream));
}

int dq_linear_fp8_dgrad(const void* dy, int64_t M, int64_t N, const uint8_t* w8, float scale, int64_t K, void* dx,
                        void* workspace, size_t workspace_bytes, dq_stream_t stream) {
  return dgrad_impl(kFmtFP8, dy, M, N, w8, nullptr, 0, scale, K, dx, workspace, workspace_bytes,
                    static_cast<cudaStream_t>(stream));
}

}  // extern "C"
