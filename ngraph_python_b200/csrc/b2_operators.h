// Helpers shared by the language-model operators (b2_embed.cu, b2_norm.cu, b2_adamw.cu, b2_heads.cu, b2_muon.cu).
#ifndef B2_OPERATORS_H
#define B2_OPERATORS_H

#include <atomic>
#include <utility>

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

// Rows of a tensor, in bytes.  Dense ones are one long row.
struct Rows {
    uintptr_t p, end;
    long long rows, width, stride;
    // of tensors of heads the heads themselves: `at_rows` x `at_heads` of `head_width` bytes (0: no such tensor)
    long long at_rows = 0, at_heads = 0, row_stride = 0, head_stride = 0, head_width = 0;
};
template <typename T>
inline Rows rows_at(const T* p, long long rows, long long width, long long stride) {
    const long long size = sizeof(T);
    const uintptr_t at = (uintptr_t)p;
    if (!p || rows <= 0 || width <= 0) return {0, 0, 0, 0, 0};
    if (rows == 1 || stride == width) return {at, at + size * rows * width, 1, size * rows * width, size * rows * width};
    return {at, at + size * ((rows - 1) * stride + width), rows, size * width, size * stride};
}

// Whether two tensors that lie among one another have memory in common.  Their rows may lie side by side, and heads of one between
// those of the other.
inline bool meet(Rows a, Rows b) {
    if (a.rows > b.rows) std::swap(a, b);
    const long long ahead = (long long)b.p - (long long)a.p;     // where b begins, seen from a
    const auto below = [](long long x, long long y) { return x / y - (x % y < 0); };
    if (a.stride == b.stride) {
        // row i of a and row j of b meet where (i - j) stride lies between ahead - a.width and ahead + b.width
        const long long least = below(ahead - a.width, a.stride) + 1, d = least > 1 - b.rows ? least : 1 - b.rows;
        if (d >= a.rows || d * a.stride >= ahead + b.width) return false;
        if (!a.at_heads || !b.at_heads) return true;
    }
    const auto alike = [](long long x, long long y, long long of_x, long long of_y) { return x == 1 || y == 1 || of_x == of_y; };
    if (a.at_heads && b.at_heads && alike(a.at_rows, b.at_rows, a.row_stride, b.row_stride) && alike(a.at_heads, b.at_heads, a.head_stride, b.head_stride)) {
        // the same at every distance that two heads have
        const long long by_row = a.at_rows > 1 ? a.row_stride : b.at_rows > 1 ? b.row_stride : 1, by_head = a.at_heads > 1 ? a.head_stride : b.head_stride;
        for (long long e = 1 - b.at_heads; e < a.at_heads; ++e) {
            const long long from = ahead - e * by_head, least = below(from - a.head_width, by_row) + 1, d = least > 1 - b.at_rows ? least : 1 - b.at_rows;
            if (d < a.at_rows && d * by_row < from + b.head_width) return true;
        }
        return false;
    }
    if (a.stride == b.stride) return true;
    for (long long i = 0; i < a.rows; ++i) {
        // the first row of b that does not end before row i of a begins
        const long long from = i * a.stride - ahead, least = below(from - b.width, b.stride) + 1, j = least > 0 ? least : 0;
        if (j < b.rows && j * b.stride < from + a.width) return true;
    }
    return false;
}

// Blocks write in any order: results have memory of their own.
inline int check_apart(const Rows* written, int count, const Rows* read, int reads, const char* what) {
    const auto apart = [](const Rows& a, const Rows& b) { return a.end <= b.p || b.end <= a.p; };
    for (int i = 0; i < count; ++i) {
        const Rows& w = written[i];
        if (!w.p) continue;
        for (int k = 0; k < i; ++k)
            if (!apart(w, written[k])) {
                B2_REQUIRE(w.p != written[k].p, "two results of the %s lie in one place", what);
                B2_REQUIRE(!meet(w, written[k]), "two results of the %s overlap", what);
            }
        for (int k = 0; k < reads; ++k)
            if (!apart(w, read[k])) {
                B2_REQUIRE(w.p != read[k].p, "a result of the %s lies in the place of an operand", what);
                B2_REQUIRE(!meet(w, read[k]), "a result of the %s overlaps an operand", what);
            }
    }
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
