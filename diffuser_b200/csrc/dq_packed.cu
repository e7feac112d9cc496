// dq_packed.cu -- include/dq_packed.h: one array of 8-byte words instead of an
// argument list.  A ctypes call converts each argument by itself (24 of them:
// 6.4 us on the host, of the 12 us that a small adapter_add took); one packed
// string of them costs 1.5 us in all.
#include <cstdint>
#include <cstring>
#include <type_traits>
#include <utility>

#include "../../include/dq_packed.h"

namespace dq {
namespace {

template <typename T>
T argument(const void* words, size_t i) {
  const char* at = static_cast<const char*>(words) + 8 * i;
  if constexpr (std::is_floating_point_v<T>) {
    double v;
    std::memcpy(&v, at, 8);
    return static_cast<T>(v);
  } else {
    int64_t v;
    std::memcpy(&v, at, 8);
    if constexpr (std::is_pointer_v<T>)
      return reinterpret_cast<T>(static_cast<uintptr_t>(v));
    else
      return static_cast<T>(v);
  }
}

template <typename... A, size_t... I>
int unpack(int (*entry)(A...), const void* words, std::index_sequence<I...>) {
  return entry(argument<A>(words, I)...);
}
template <typename... A>
int call(int (*entry)(A...), const void* words) {
  return words == nullptr ? DQ_ERR_ARG : unpack(entry, words, std::index_sequence_for<A...>());
}

}  // namespace
}  // namespace dq

extern "C" {

int dq_adapter_add_packed(const void* words) { return dq::call(dq_adapter_add, words); }
int dq_adapter_backward_packed(const void* words) { return dq::call(dq_adapter_backward, words); }
int dq_checkpoint_pack_packed(const void* words) { return dq::call(dq_checkpoint_pack, words); }
int dq_checkpoint_unpack_packed(const void* words) { return dq::call(dq_checkpoint_unpack, words); }
int dq_linear_nf4_dgrad_packed(const void* words) { return dq::call(dq_linear_nf4_dgrad, words); }
int dq_linear_fp8_dgrad_packed(const void* words) { return dq::call(dq_linear_fp8_dgrad, words); }
int dq_gated_norm_packed(const void* words) { return dq::call(dq_gated_norm, words); }
int dq_gated_norm_backward_packed(const void* words) { return dq::call(dq_gated_norm_backward, words); }

}  // extern "C"
