// dq_internal.h -- what the translation units of the library share besides the
// public headers (none of it is exported API).
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

namespace dq {

// Facts of the current device; DQ_ERR_ARCH unless it is an sm_100.
int device_sms(int* sms);

// Device address of the current device's kernel error word (dq_device_error
// reads and clears it): kernels of other translation units record bits there.
// The first call on a device looks it up; it is cached from then on.
int error_word(unsigned int** word);

// Bits of the error word: a bounded wait expired; an index on the device was out
// of range.
enum : unsigned int { kErrTimeout = 5u, kErrIndex = 10u };

// y[M, N] (row stride ldy) = x[M, K] . w[N, K]^T, all bf16, on the CTA-pair
// GEMM without its decode.  K % 8 == 0, x / w 16-byte aligned.
int bf16_gemm(const void* x, int64_t M, int64_t K, const void* w, int64_t N, void* y, int64_t ldy,
              cudaStream_t st);

// Tensor map of a row-major bf16 matrix [outer, inner], rows row_bytes apart, in
// boxes of [box_outer, 64] elements with the 128-byte swizzle (map: a
// CUtensorMap); false if the driver refuses it.
bool bf16_tile_map(void* map, const void* base, uint64_t inner, uint64_t outer, uint64_t row_bytes,
                   uint32_t box_outer);

}  // namespace dq
