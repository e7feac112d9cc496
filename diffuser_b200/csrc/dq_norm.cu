// dq_norm.cu -- host side of dq_gated_norm and its backward pass
// (include/dq_dit.h): argument validation and launches.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "../../include/dq_dit.h"
#include "dq_internal.h"
#include "dq_launch.h"
#include "dq_norm.cuh"

namespace dq {
namespace {

inline const __nv_bfloat16* bf(const void* p) { return static_cast<const __nv_bfloat16*>(p); }

// An output in the place of an operand has its rows.
bool same_rows(const void* out, int64_t ld_out, const void* in, int64_t ld_in) { return out != in || ld_out == ld_in; }

bool stride_ok(int64_t ld, int D) { return ld >= D && ld % 4 == 0; }

int shape_ok(int64_t T, int S, int D) {
  return T < 0 || S <= 0 || D <= 0 || D % 4 != 0 || D > 8192 || T > INT32_MAX || T % S != 0 ? DQ_ERR_SHAPE : DQ_OK;
}

bool norms_ok(int post, int pre, const void* post_w) {
  return post >= kNormNone && post <= kNormLayer && (pre == kNormRms || pre == kNormLayer) &&
         (post_w == nullptr || post != kNormNone);
}

// CTAs per batch element: what fills `slots` over all elements, at least `least`
// rows each (a CTA's factors and, backward, its column sums are a fixed cost).
int chunks_of(int64_t B, int S, int64_t slots, int least) {
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(slots / std::max<int64_t>(1, B), ceil_div(S, least))));
}
int64_t backward_slots(int D, int sms) {
  return static_cast<int64_t>(sms) * (D <= 2048 ? norm_grad_ctas(128, 4) : D <= 4096 ? norm_grad_ctas(128, 8) : 1);
}

// Shared-memory opt-in of a kernel and its resident CTAs per SM, once per
// kernel and device.
struct KernelInfo {
  std::atomic<int> per_sm[kMaxDevices];  // 0: not set up
};
template <typename K>
int set_up(K kern, int threads, size_t most, KernelInfo& info, int* per_sm) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return DQ_ERR_CUDA;
  int n = info.per_sm[dev].load(std::memory_order_acquire);
  if (n == 0) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most)) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, most) != cudaSuccess || n < 1)
      return DQ_ERR_LAUNCH;
    info.per_sm[dev].store(n, std::memory_order_release);
  }
  *per_sm = n;
  return DQ_OK;
}

template <int NPT, bool OPS, bool FULL>
int launch_forward_npt(NormArgs a, int64_t B, int sms, cudaStream_t st) {
  static KernelInfo info;
  const size_t per_feature = kNormAhead * 4 + (OPS ? 0 : 12);
  int per_sm = 1;
  const int rc = set_up(gated_norm_kernel<NPT, OPS, FULL>, kNormThreads, per_feature * NPT * kNormThreads * 4,
                        info, &per_sm);
  if (rc != DQ_OK) return rc;
  a.chunks = chunks_of(B, a.S, static_cast<int64_t>(sms) * per_sm, 1);
  gated_norm_kernel<NPT, OPS, FULL><<<static_cast<unsigned>(B * a.chunks), kNormThreads, per_feature * a.D, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? DQ_OK : DQ_ERR_LAUNCH;
}

template <int NPT, bool OPS>
int launch_forward_runs(const NormArgs& a, int64_t B, int sms, cudaStream_t st) {
  return a.D == 4 * NPT * kNormThreads ? launch_forward_npt<NPT, OPS, true>(a, B, sms, st)
                                       : launch_forward_npt<NPT, OPS, false>(a, B, sms, st);
}

template <bool OPS>
int launch_forward(const NormArgs& a, int64_t B, int sms, cudaStream_t st) {
  switch ((a.D / 4 + kNormThreads - 1) / kNormThreads) {
    case 1: return launch_forward_runs<1, OPS>(a, B, sms, st);
    case 2: return launch_forward_runs<2, OPS>(a, B, sms, st);
    case 3: return launch_forward_runs<3, OPS>(a, B, sms, st);
    case 4: return launch_forward_runs<4, OPS>(a, B, sms, st);
    case 5:
    case 6: return launch_forward_runs<6, OPS>(a, B, sms, st);
  }
  return launch_forward_runs<8, OPS>(a, B, sms, st);
}

template <int THREADS, int NPT, bool FULL>
int launch_backward_npt(const NormGradArgs& a, int64_t B, cudaStream_t st) {
  static KernelInfo info;
  constexpr size_t kPerFeature = kNormGradAhead * 8 + 8;
  int per_sm = 1;
  const int rc = set_up(gated_norm_backward_kernel<THREADS, NPT, FULL>, THREADS, kPerFeature * THREADS * NPT * 4,
                        info, &per_sm);
  if (rc != DQ_OK) return rc;
  gated_norm_backward_kernel<THREADS, NPT, FULL>
      <<<static_cast<unsigned>(B * a.chunks), THREADS, kPerFeature * a.D, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? DQ_OK : DQ_ERR_LAUNCH;
}

template <int THREADS, int NPT>
int launch_backward(const NormGradArgs& a, int64_t B, cudaStream_t st) {
  return a.D == 4 * NPT * THREADS ? launch_backward_npt<THREADS, NPT, true>(a, B, st)
                                  : launch_backward_npt<THREADS, NPT, false>(a, B, st);
}

}  // namespace
}  // namespace dq

using namespace dq;

extern "C" {

int dq_gated_norm(const void* x, int64_t ld_x, const void* y, int64_t ld_y, int64_t T, int S, int D,
                  const void* gate, int64_t ld_gate, const void* scale, const void* shift, int64_t ld_mod,
                  const void* post_weight, const void* pre_weight, int post, int pre, float residual_scale, float eps,
                  int rounding, void* s, int64_t ld_s, void* h, int64_t ld_h, dq_stream_t stream) {
  int rc = shape_ok(T, S, D);
  if (rc != DQ_OK) return rc;
  if (!norms_ok(post, pre, post_weight) || rounding < DQ_ROUND_ONCE || rounding > DQ_ROUND_OPS) return DQ_ERR_ARG;
  if (T == 0) return DQ_OK;
  if (x == nullptr || y == nullptr || s == nullptr || h == nullptr) return DQ_ERR_ARG;
  if (!stride_ok(ld_x, D) || !stride_ok(ld_y, D) || !stride_ok(ld_s, D) || !stride_ok(ld_h, D) ||
      (gate != nullptr && !stride_ok(ld_gate, D)) ||
      ((scale != nullptr || shift != nullptr) && !stride_ok(ld_mod, D)))
    return DQ_ERR_SHAPE;
  for (const void* p : {x, y, gate, scale, shift, post_weight, pre_weight, static_cast<const void*>(s),
                        static_cast<const void*>(h)})
    if (!aligned(p, 8)) return DQ_ERR_ALIGN;
  // in place row by row, or rows of another stride are written before they are read
  if (s == h) return DQ_ERR_ARG;
  if (!same_rows(s, ld_s, x, ld_x) || !same_rows(s, ld_s, y, ld_y) || !same_rows(h, ld_h, x, ld_x) ||
      !same_rows(h, ld_h, y, ld_y))
    return DQ_ERR_SHAPE;
  int sms = 0;
  if ((rc = device_sms(&sms)) != DQ_OK) return rc;
  const NormArgs a = {bf(x), bf(y), bf(gate), bf(scale), bf(shift), bf(post_weight), bf(pre_weight),
                      static_cast<__nv_bfloat16*>(s), static_cast<__nv_bfloat16*>(h), ld_x, ld_y, ld_gate, ld_mod,
                      ld_s, ld_h, S, D, post, pre, 0, residual_scale, eps};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return rounding == DQ_ROUND_OPS ? launch_forward<true>(a, T / S, sms, st) : launch_forward<false>(a, T / S, sms, st);
}

size_t dq_gated_norm_backward_workspace(int64_t T, int S, int D) {
  int sms = 0;
  if (shape_ok(T, S, D) != DQ_OK || T == 0 || device_sms(&sms) != DQ_OK) return 0;
  const int64_t B = T / S;
  return static_cast<size_t>(B) * chunks_of(B, S, backward_slots(D, sms), 4) * 3 * D * sizeof(float);
}

int dq_gated_norm_backward(const void* ds, int64_t ld_ds, const void* dh, int64_t ld_dh, const void* s, int64_t ld_s,
                           const void* y, int64_t ld_y, int64_t T, int S, int D, const void* gate, int64_t ld_gate,
                           const void* scale, int64_t ld_mod, const void* post_weight, const void* pre_weight, int post,
                           int pre, float residual_scale, float eps, void* dx, int64_t ld_dx, void* dy, int64_t ld_dy,
                           float* dgate, float* dscale, float* dshift, float* dpost_weight, float* dpre_weight,
                           void* workspace, size_t workspace_bytes, dq_stream_t stream) {
  int rc = shape_ok(T, S, D);
  if (rc != DQ_OK) return rc;
  if (!norms_ok(post, pre, post_weight)) return DQ_ERR_ARG;
  const int64_t B = T / S;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {  // no tokens: the weights' gradients are zeros
    for (float* p : {dpost_weight, dpre_weight})
      if (p != nullptr && cudaMemsetAsync(p, 0, static_cast<size_t>(D) * 4, st) != cudaSuccess) return DQ_ERR_CUDA;
    return DQ_OK;
  }
  if (dh == nullptr || s == nullptr || y == nullptr || dx == nullptr || dy == nullptr) return DQ_ERR_ARG;
  if ((ds != nullptr && !stride_ok(ld_ds, D)) || !stride_ok(ld_dh, D) || !stride_ok(ld_s, D) || !stride_ok(ld_y, D) ||
      !stride_ok(ld_dx, D) || !stride_ok(ld_dy, D) || (gate != nullptr && !stride_ok(ld_gate, D)) ||
      (scale != nullptr && !stride_ok(ld_mod, D)))
    return DQ_ERR_SHAPE;
  for (const void* p : {ds, dh, s, y, gate, scale, post_weight, pre_weight, static_cast<const void*>(dx),
                        static_cast<const void*>(dy)})
    if (!aligned(p, 8)) return DQ_ERR_ALIGN;
  for (const float* p : {dgate, dscale, dshift, dpost_weight, dpre_weight})
    if (!aligned(p, 4)) return DQ_ERR_ALIGN;
  if (dx == dy) return DQ_ERR_ARG;
  for (const void* out : {static_cast<const void*>(dx), static_cast<const void*>(dy)}) {
    const int64_t ld = out == dx ? ld_dx : ld_dy;
    if (!same_rows(out, ld, ds, ld_ds) || !same_rows(out, ld, dh, ld_dh) || !same_rows(out, ld, s, ld_s) ||
        !same_rows(out, ld, y, ld_y))
      return DQ_ERR_SHAPE;
  }
  int sms = 0;
  if ((rc = device_sms(&sms)) != DQ_OK) return rc;
  const int chunks = chunks_of(B, S, backward_slots(D, sms), 4);
  if (workspace == nullptr || !aligned(workspace, 16) ||
      workspace_bytes < static_cast<size_t>(B) * chunks * 3 * D * sizeof(float))
    return DQ_ERR_WORKSPACE;
  NormGradArgs a = {bf(ds), bf(dh), bf(s), bf(y), bf(gate), bf(scale), bf(post_weight), bf(pre_weight),
                    static_cast<__nv_bfloat16*>(dx), static_cast<__nv_bfloat16*>(dy), static_cast<float*>(workspace),
                    ld_ds, ld_dh, ld_s, ld_y, ld_gate, ld_mod, ld_dx, ld_dy, S, D, post, pre,
                    chunks, residual_scale, eps};
  const int runs = D / 4;
  rc = runs <= 256    ? launch_backward<128, 2>(a, B, st)
       : runs <= 512  ? launch_backward<128, 4>(a, B, st)
       : runs <= 768  ? launch_backward<128, 6>(a, B, st)
       : runs <= 1024 ? launch_backward<128, 8>(a, B, st)
                      : launch_backward<256, 8>(a, B, st);
  if (rc != DQ_OK) return rc;
  NormReduceArgs q = {a.part, a.gate, a.scale, a.post_w, a.pre_w, dgate, dscale, dshift, dpost_weight, dpre_weight,
                      ld_gate, ld_mod, static_cast<int>(B), chunks, D, residual_scale};
  if (dgate != nullptr || dscale != nullptr || dshift != nullptr || dpost_weight != nullptr || dpre_weight != nullptr)
    // it may start while the last rows are on their way out, and waits for them
    return launch(gated_norm_reduce_kernel, dim3(static_cast<unsigned>(ceil_div(D, 32))), 32 * kReduceWarps, 0, st, true,
                  dim3(1), q);
  return DQ_OK;
}

}  // extern "C"
