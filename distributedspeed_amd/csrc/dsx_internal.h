// dsx_internal.h -- what the library's translation units share on the host.
#ifndef DSX_INTERNAL_H_
#define DSX_INTERNAL_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "dsx.h"

namespace dsxi {

// Records the message dsx_last_error() returns and passes `code` through.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int fail(int code, const char* fmt, ...);
__attribute__((visibility("hidden"))) int launch_status(const char* what);

inline hipStream_t as_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }
inline bool is16(int dt) { return dt == DSX_F16 || dt == DSX_BF16; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

}  // namespace dsxi

#endif  // DSX_INTERNAL_H_
