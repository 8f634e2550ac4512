// lsk_call: entry points by number, their arguments as 64-bit words.  A binding that converts each argument by itself
// spends a good part of a small launch on it (ctypes, the 28 of lsk_kv4_attn: 1.1 us against 0.25 for one packed array).
// Host code only.
#include <string.h>
#include <utility>
#include "lsk_common.h"
#include "../include/lsk.h"

namespace {

template <typename T>
T word(const int64_t* w) {
  if constexpr (std::is_pointer<T>::value) return (T)(uintptr_t)*w;
  else if constexpr (std::is_floating_point<T>::value) {
    double d;
    memcpy(&d, w, sizeof d);
    return (T)d;
  } else return (T)*w;
}

template <typename... A, size_t... I>
int call(int (*f)(A...), const int64_t* w, std::index_sequence<I...>) { return f(word<A>(w + I)...); }

template <typename... A>
int call(int (*f)(A...), int n, const int64_t* w) {
  LSK_REQUIRE(n == (int)sizeof...(A) && w, LSK_EARG, "lsk_call: %d arguments for an entry of %d", n, (int)sizeof...(A));
  return call(f, w, std::index_sequence_for<A...>());
}

}  // namespace

extern "C" int lsk_call(int entry, int n_args, const int64_t* args) {
  switch (entry) {
    case LSK_CALL_KV4_APPEND: return call(lsk_kv4_append, n_args, args);
    case LSK_CALL_KV4_READ: return call(lsk_kv4_read, n_args, args);
    case LSK_CALL_KV4_ATTN: return call(lsk_kv4_attn, n_args, args);
    case LSK_CALL_QK_NORM_ROPE: return call(lsk_qk_norm_rope, n_args, args);
    case LSK_CALL_QUANT_ROWS_I8: return call(lsk_quant_rows_i8, n_args, args);
    case LSK_CALL_GEMM_I8: return call(lsk_gemm_i8, n_args, args);
  }
  LSK_REQUIRE(false, LSK_EARG, "lsk_call: no entry %d", entry);
}
