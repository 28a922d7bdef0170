// What the translation units of libmt_flce.so share on the host side: the
// thread's last error and the check of a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/mt_flce.h"

namespace mtf {

// Records the thread's last error (mt_flce_last_error) and returns `code`.
int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// MT_OK, or MT_ERR_HIP if the launch just made failed (or is made to look so
// by the test hook MT_FLCE_TEST_FAIL_LAUNCH).
int check_launch(const char* what);

inline int esize(int dtype) {
  return dtype == MT_DTYPE_BF16 ? 2 : (dtype == MT_DTYPE_F32 ? 4 : 0);
}
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
constexpr int64_t kMaxRows = INT32_MAX - 1024;  // row numbers, plus a block, in 32 bits

}  // namespace mtf

#define MT_TRY(expr)             \
  do {                           \
    int _rc = (expr);            \
    if (_rc != MT_OK) return _rc; \
  } while (0)
