// What the translation units of liboeq_amd.so share for reporting errors: the message of the calling thread's last
// failure (oeq_last_error) and the two ways to leave one.
#ifndef OEQ_ERROR_H
#define OEQ_ERROR_H

#include "oeq_amd.h"

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <string>

namespace oeq_internal {

inline thread_local std::string g_error;

inline int fail(int code, const char* fmt, ...) {
    char buf[2048];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    g_error = buf;
    return code;
}

}  // namespace oeq_internal

#define HIP_TRY(expr)                                                                                 \
    do {                                                                                              \
        hipError_t e_ = (expr);                                                                       \
        if (e_ != hipSuccess)                                                                         \
            return oeq_internal::fail(OEQ_ERR_HIP, "%s failed: %s", #expr, hipGetErrorString(e_));    \
    } while (0)

#endif
