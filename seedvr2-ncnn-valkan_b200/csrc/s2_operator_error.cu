// s2_operator_device_error: what the channels-last operators report when a bounded wait gives up in a call
// without an error word. A device variable rather than an allocation: it is there before the first call,
// which may be inside a stream capture.
#include <cuda_runtime.h>

#include <atomic>

#include "s2_b200.h"
#include "s2_internal.h"
#include "s2_operator_error.h"

namespace {

__device__ int32_t g_word;
std::atomic<int32_t *> g_words[64];

}  // namespace

namespace s2 {

int32_t *operator_error_word()
{
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return nullptr;
    }
    int32_t *word = g_words[dev].load(std::memory_order_acquire);
    if (!word) {
        void *p = nullptr;
        if (cudaGetSymbolAddress(&p, g_word) != cudaSuccess) {
            cudaGetLastError();
            return nullptr;
        }
        word = static_cast<int32_t *>(p);
        g_words[dev].store(word, std::memory_order_release);
    }
    return word;
}

}  // namespace s2

extern "C" s2_status s2_operator_device_error(int *code)
{
    s2::clear_error();
    if (code) *code = 0;
    int32_t *word = s2::operator_error_word();
    int32_t h = 0;
    // cleared before this returns: what the caller runs next may report again
    if (!word || cudaDeviceSynchronize() != cudaSuccess || cudaMemcpy(&h, word, 4, cudaMemcpyDeviceToHost) != cudaSuccess ||
        (h != 0 && (cudaMemset(word, 0, 4) != cudaSuccess || cudaDeviceSynchronize() != cudaSuccess)))
        return s2::set_error(S2_INFERENCE_FAILED, "s2_operator_device_error: device failure: %s",
                             cudaGetErrorString(cudaGetLastError()));
    if (code) *code = h;
    if (h != 0)
        return s2::set_error(S2_INFERENCE_FAILED, "a channels-last operator gave up a wait on the device (code %d)", h);
    return S2_OK;
}
