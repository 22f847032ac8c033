// The device status word of the training operators. Their kernels wait with a limit and run without the host waiting for them, so what
// a wait that ran out has to say stays here until it is read and cleared (tffn_train_status).
#include "train.h"
#include <mutex>

namespace tffn {

static __device__ int g_train_status;  // in host code a handle for the runtime

int* train_status_word(int device) {
    static std::mutex mu;
    static int* known[64] = {nullptr};
    if (device < 0 || device >= 64) return nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (!known[device]) {
        void* p = nullptr;
        if (cudaGetSymbolAddress(&p, g_train_status) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        known[device] = (int*)p;
    }
    return known[device];
}

}  // namespace tffn
