// What the C ABI's host files share: error codes with their message, checks, workspace layout.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/psgdk.h"

namespace psgdk {
int set_error(int code, const char* msg);

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}
int hip_check(hipError_t e, const char* what) {
  return e == hipSuccess ? PSGDK_OK : fail(PSGDK_EHIP, "%s: %s", what, hipGetErrorString(e));
}
#define PSGDK_TRY(expr)              \
  do {                               \
    const int _rc = (expr);          \
    if (_rc != PSGDK_OK) return _rc; \
  } while (0)

int check_dt(int dt, const char* name) {
  if (dt != PSGDK_F32 && dt != PSGDK_BF16) return fail(PSGDK_EINVAL, "%s = %d", name, dt);
  return PSGDK_OK;
}
int check_size(int64_t v, int64_t lo, int64_t hi, const char* name) {
  if (v < lo || v > hi)
    return fail(PSGDK_ESHAPE, "%s = %lld: must be in %lld..%lld", name, (long long)v, (long long)lo, (long long)hi);
  return PSGDK_OK;
}
size_t esize(int dt) { return dt == PSGDK_BF16 ? 2 : 4; }

// Bump allocator over the caller's workspace; with base == nullptr it only measures.
struct Ws {
  char* base;
  size_t off = 0;
  explicit Ws(void* b) : base(static_cast<char*>(b)) {}
  template <typename T>
  T* take(size_t count) {
    off = (off + 255) & ~size_t(255);
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += count * sizeof(T);
    return p;
  }
};

}  // namespace
}  // namespace psgdk
