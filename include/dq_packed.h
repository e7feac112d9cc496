/* dq_packed.h -- entry points for bindings that pay for every argument they
 * convert (same library as dq_linear.h).
 *
 * dq_<name>_packed(words) is dq_<name>(...): words holds its arguments in
 * order, 8 bytes each in host memory -- pointers and integers as int64, floats
 * as double.  Nothing is kept of the array after the call. */
#ifndef DQ_PACKED_H
#define DQ_PACKED_H

#include "dq_adapter.h"
#include "dq_dit.h"

#ifdef __cplusplus
extern "C" {
#endif

int dq_adapter_add_packed(const void* words);
int dq_adapter_backward_packed(const void* words);
int dq_checkpoint_pack_packed(const void* words);
int dq_checkpoint_unpack_packed(const void* words);
int dq_linear_nf4_dgrad_packed(const void* words);
int dq_linear_fp8_dgrad_packed(const void* words);
int dq_gated_norm_packed(const void* words);
int dq_gated_norm_backward_packed(const void* words);

#ifdef __cplusplus
}
#endif

#endif /* DQ_PACKED_H */
