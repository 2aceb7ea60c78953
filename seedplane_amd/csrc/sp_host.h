// Host-side plumbing shared by the library's translation units: the exception the C ABI turns into a status and a message,
// argument checks, HIP status checks, device allocations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

#include "../../include/seedplane_hip.h"

// The message sp_last_error() returns on this thread.
__attribute__((visibility("hidden"))) std::string &sp_call_error();

namespace {

struct Fail {
    int code;
    std::string msg;
};

#define HIPCHK(expr)                                                                                     \
    do {                                                                                                 \
        hipError_t _e = (expr);                                                                          \
        if (_e != hipSuccess)                                                                            \
            throw Fail{SP_EHIP, std::string(#expr) + ": " + hipGetErrorString(_e)};                      \
    } while (0)

[[maybe_unused]] inline void require(bool ok, int code, const std::string &msg) {
    if (!ok) throw Fail{code, msg};
}
// A literal message builds its string only on failure (per-column checks run on every call).
[[maybe_unused]] inline void require(bool ok, int code, const char *msg) {
    if (!ok) throw Fail{code, msg};
}

template <class T>
T *dev_alloc(size_t count, uint64_t *acct = nullptr) {
    void *p = nullptr;
    if (count == 0) count = 1;
    hipError_t e = hipMalloc(&p, count * sizeof(T));
    if (e != hipSuccess) throw Fail{SP_ENOMEM, "hipMalloc of " + std::to_string(count * sizeof(T)) + " bytes failed: " + hipGetErrorString(e)};
    if (acct) *acct += count * sizeof(T);
    return (T *)p;
}
[[maybe_unused]] inline void dev_free(void *p) {
    if (p) (void)hipFree(p);
}

}  // namespace
