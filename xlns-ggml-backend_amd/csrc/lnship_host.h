// What the host sides of the kernel files share: errors and the per-device
// state that lnship_init sets up (both defined in lnship_kernels.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <vector>

#include "lnship_device.h"

namespace lnship {

constexpr int k_block = 256;
constexpr int k_max_devices = 64;

// records the calling thread's error (fmt has one %s, for what); returns code
#define LNSHIP_HIDDEN __attribute__((visibility("hidden")))
LNSHIP_HIDDEN int fail(int code, const char *fmt, const char *what = "");
LNSHIP_HIDDEN int hip_fail(hipError_t e, const char *where);

#define LNSHIP_HIP(call)                                          \
    do {                                                          \
        hipError_t e_ = (call);                                   \
        if (e_ != hipSuccess) return hip_fail(e_, #call);         \
    } while (0)

struct device_state {
    bool ready = false;
    int cus = 0;   // compute units
    dev_tables T{};
    void *scratch = nullptr;   // grow-only
    size_t scratch_size = 0;
    std::vector<void *> retired;   // outgrown scratch blocks, kept for captured graphs
    void *fixed_scratch = nullptr;  // this device's copy of `scratch` (below), from hipGetSymbolAddress
    // index check (rows, positions, pages): [0] set to 1 by the first
    // out-of-range index since the last lnship_index_error, [1] that index
    unsigned long long *index_err = nullptr;
};

LNSHIP_HIDDEN int current_device(int *dev);
// the current device's state; null, with the error recorded, before lnship_init
LNSHIP_HIDDEN device_state *state();

}  // namespace lnship
