// moe_host.cpp -- the C ABI's per-thread error message (moe_host.h).

#include "moe_host.h"

#include <cstdarg>
#include <cstdio>

namespace moe {
namespace host {

namespace {
thread_local char g_last_error[512] = "";
}

moe_status fail(moe_status st, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
    va_end(ap);
    return st;
}

moe_status ok() {
    g_last_error[0] = '\0';
    return MOE_OK;
}

moe_status hip_fail(hipError_t err, const char* what) {
    return fail(MOE_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

const char* last_error() { return g_last_error; }

}  // namespace host
}  // namespace moe
