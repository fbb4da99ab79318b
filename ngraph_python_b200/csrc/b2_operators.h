// Helpers shared by the language-model operators (b2_embed.cu, b2_norm.cu, b2_adamw.cu).
#ifndef B2_OPERATORS_H
#define B2_OPERATORS_H

#include <atomic>

#include "b2_common.h"

namespace b2 {

constexpr int kSms = 148;

// Launches go to the current device.  A result that lies on another one, or on the host, is refused: the kernel would
// fault, or write across the link.  Operands may also lie in page-locked host memory.  (50 ns an address, and 25 for the
// device, which is looked up once in a call.)
class Memory {
  public:
    int find_device() {
        B2_CUDA(cudaGetDevice(&now_));
        return B2_OK;
    }
    int written(const void* out, const char* what) const {
        cudaPointerAttributes a;
        B2_CUDA(cudaPointerGetAttributes(&a, out));
        B2_REQUIRE(a.type == cudaMemoryTypeDevice || a.type == cudaMemoryTypeManaged, "%s is not device memory", what);
        B2_REQUIRE(a.type != cudaMemoryTypeDevice || a.device == now_, "%s lies on device %d, the current device is %d", what, a.device, now_);
        return B2_OK;
    }
    int read(const void* in, const char* what) {
        if (!in) return B2_OK;
        cudaPointerAttributes a;
        B2_CUDA(cudaPointerGetAttributes(&a, in));
        B2_REQUIRE(a.type != cudaMemoryTypeUnregistered, "%s is not memory that the device reads", what);
        B2_REQUIRE(a.type != cudaMemoryTypeDevice || a.device == now_, "%s lies on device %d, the current device is %d", what, a.device, now_);
        elsewhere = elsewhere || a.type != cudaMemoryTypeDevice;
        return B2_OK;
    }
    bool elsewhere = false;             // an operand is not device memory

  private:
    int now_ = 0;
};

// Blocks write in any order: a dense result has no memory in common with an operand.
inline bool overlap(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
    return a && b && a_bytes && b_bytes && (uintptr_t)a < (uintptr_t)b + b_bytes &&
           (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// More than 48 KB of dynamic shared memory is asked for once per kernel and device.
inline int allow_shared(const void* kernel, int bytes, std::atomic<unsigned long long>* done) {
    int now = 0;
    B2_CUDA(cudaGetDevice(&now));
    const unsigned long long bit = 1ull << (now & 63);
    if (done->load(std::memory_order_relaxed) & bit) return B2_OK;
    B2_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done->fetch_or(bit, std::memory_order_relaxed);
    return B2_OK;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace b2

#define B2_CHECK(call)              \
    do {                            \
        int rc__ = (call);          \
        if (rc__ < 0) return rc__;  \
    } while (0)

#endif  // B2_OPERATORS_H
