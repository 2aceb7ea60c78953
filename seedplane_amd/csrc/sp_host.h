// Host-side plumbing shared by the library's translation units: the exception the C ABI turns into a status and a message,
// argument checks, HIP status checks, device allocations.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <new>
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

// What a C entry does: no exception passes it.
template <class F>
int guarded(F &&fn) {
    try {
        fn();
        return SP_OK;
    } catch (const Fail &f) {
        sp_call_error() = f.msg;
        return f.code;
    } catch (const std::bad_alloc &) {
        sp_call_error() = "out of host memory";
        return SP_ENOMEM;
    } catch (const std::exception &ex) {
        sp_call_error() = ex.what();
        return SP_EHIP;
    }
}

}  // namespace
