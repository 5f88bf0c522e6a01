// Argument checks that the entry points share.  They run before any HIP call.
#pragma once
#include "axn_internal.h"

namespace axn {
namespace {

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }

#define REQUIRE(cond, code, ...)   \
  do {                             \
    if (!(cond)) {                 \
      set_error(__VA_ARGS__);      \
      return (code);               \
    }                              \
  } while (0)

bool known_dtype(int dt) { return dt == AXN_BF16 || dt == AXN_F16 || dt == AXN_F32; }

int check_list(const char* name, const void* const* h_ptrs, const char* what,
               const int64_t* h_sizes, int64_t n, int elem_size) {
  for (int64_t i = 0; i < n; ++i) {
    if (h_sizes[i] == 0) continue;
    REQUIRE(h_ptrs[i] != nullptr, AXN_EINVAL, "%s: %s[%lld] is null", name, what,
            (long long)i);
    REQUIRE(((uintptr_t)h_ptrs[i] % (uintptr_t)elem_size) == 0, AXN_EALIGN,
            "%s: %s[%lld] is not aligned to its element size", name, what,
            (long long)i);
  }
  return AXN_OK;
}

int check_sizes(const char* name, const int64_t* h_sizes, int64_t n) {
  REQUIRE(n >= 0, AXN_EINVAL, "%s: negative tensor count", name);
  REQUIRE(n == 0 || h_sizes != nullptr, AXN_EINVAL, "%s: null size array", name);
  for (int64_t i = 0; i < n; ++i)
    REQUIRE(h_sizes[i] >= 0, AXN_EINVAL, "%s: sizes[%lld] is negative", name,
            (long long)i);
  return AXN_OK;
}

}  // namespace
}  // namespace axn
