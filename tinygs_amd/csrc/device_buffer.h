// Grow-only device scratch of the C ABI's handles.
#pragma once

#include "status.h"

namespace tgs {

struct DevBuf {
    void* p = nullptr;
    size_t bytes = 0;
    template <typename T>
    T* as() const { return (T*)p; }
};

// Grow-only device allocation. A grown buffer is released only after the
// stream has drained, so kernels of earlier calls never see freed memory.
inline int ensure(DevBuf& b, size_t bytes, hipStream_t s) {
    if (bytes <= b.bytes && b.p) return TGS_OK;
    if (b.p) {
        TGS_HIP(hipStreamSynchronize(s));
        TGS_HIP(hipFree(b.p));
        b.p = nullptr;
        b.bytes = 0;
    }
    size_t nb = bytes + bytes / 4 + 256;
    TGS_HIP(hipMalloc(&b.p, nb));
    b.bytes = nb;
    return TGS_OK;
}

inline void release(DevBuf& b) {
    if (b.p) (void)hipFree(b.p);
    b.p = nullptr;
    b.bytes = 0;
}

}  // namespace tgs
