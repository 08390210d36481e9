// Status texts and the reports of kernels: two ints of pinned host memory per device, written by the kernel that sees
// a problem and read by the host without waiting.
#include <mutex>

#include "train_common.h"

namespace i6train {
namespace {
constexpr int kMaxDevices = 64;
std::mutex g_mutex;
int* g_slots[kMaxDevices];
}  // namespace

int* status_slot() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
    std::lock_guard<std::mutex> lock(g_mutex);
    if (!g_slots[dev]) {
        void* p = nullptr;
        if (hipHostMalloc(&p, 2 * sizeof(int), hipHostMallocDefault) != hipSuccess) return nullptr;
        g_slots[dev] = static_cast<int*>(p);
        g_slots[dev][0] = I6TRAIN_OK;
        g_slots[dev][1] = -1;
    }
    return g_slots[dev];
}
}  // namespace i6train

extern "C" {

const char* i6train_strerror(int code) {
    switch (code) {
        case I6TRAIN_OK: return "ok";
        case I6TRAIN_ERR_INVALID_ARGUMENT: return "invalid argument";
        case I6TRAIN_ERR_WORKSPACE_TOO_SMALL: return "workspace too small";
        case I6TRAIN_ERR_LAUNCH: return "HIP call failed";
        case I6TRAIN_ERR_TOO_LARGE: return "the problem is larger than this operator takes";
        case I6TRAIN_ERR_BAD_TARGET: return "target out of range";
        default: return "unknown status";
    }
}

int i6train_poll_status(int* code, int* seq) {
    if (!code || !seq) return I6TRAIN_ERR_INVALID_ARGUMENT;
    int* slot = i6train::status_slot();
    if (!slot) return I6TRAIN_ERR_LAUNCH;
    volatile int* s = slot;
    *code = s[0];
    *seq = s[1];
    if (*code != I6TRAIN_OK) {
        s[0] = I6TRAIN_OK;
        s[1] = -1;
    }
    return I6TRAIN_OK;
}

}  // extern "C"
