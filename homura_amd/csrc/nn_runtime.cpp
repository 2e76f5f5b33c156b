// The calling thread's failure text of libhomura_nn, and what else the shared headers leave to the library they are
// linked into (the failure functions of common.hpp).
#include <string>

#include "common.hpp"
#include "homura_nn.h"

namespace hmr {
namespace {

struct ThreadText {
    std::string text;
    const char *literal = nullptr;  // instead of the text, where nothing may be allocated
};

ThreadText &mine() {
    thread_local ThreadText state;
    return state;
}

}  // namespace

hmr_status fail(hmr_status status, std::string message) {
    ThreadText &t = mine();
    t.text = std::move(message);
    t.literal = nullptr;
    return status;
}

hmr_status fail_static(hmr_status status, const char *message) noexcept {
    mine().literal = message;
    return status;
}

const char *last_error_text() noexcept {
    const ThreadText &t = mine();
    return t.literal ? t.literal : t.text.c_str();
}

hmr_status hip_failure(hipError_t error, const char *what) noexcept {
    (void)hipGetLastError();
    const hmr_status status = error == hipErrorOutOfMemory ? HMR_OUT_OF_MEMORY : HMR_HIP_ERROR;
    const char *description = hipGetErrorString(error);
    try {
        return fail(status, std::string(what) + ": " + description);
    } catch (...) {
        return fail_static(status, description);
    }
}

// The failures a test arms belong to libhomura_rocm's entry points.
hmr_status Visit::armed_failure(const char *) noexcept { return HMR_OK; }

}  // namespace hmr

extern "C" const char *hmn_last_error(void) { return hmr::last_error_text(); }
