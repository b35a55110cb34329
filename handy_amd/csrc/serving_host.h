// Host side of the serving operators' C entries (k_paged.hip, k_draw.hip): which device a call belongs to, and whether the
// buffers it was handed are that device's memory.
#pragma once
#include "wmi_common.h"

namespace wmi {

// A call runs on its stream's device (the null stream: the calling thread's current one), whatever the current device is;
// the caller's current device is put back. Nothing here allocates, waits or throws, and all of it is allowed under capture.
class ServeCall {
public:
    explicit ServeCall(hipStream_t st) {
        if (hipGetDevice(&prev_) != hipSuccess) { (void)hipGetLastError(); return; }
        dev_ = prev_;
        if ((uintptr_t)st > 2 && hipStreamGetDevice(st, &dev_) != hipSuccess) { (void)hipGetLastError(); dev_ = -1; return; }     // 0 null, 1 legacy, 2 per-thread
        if (dev_ != prev_ && hipSetDevice(dev_) != hipSuccess) { (void)hipGetLastError(); dev_ = -1; }
    }
    ~ServeCall() { if (dev_ >= 0 && dev_ != prev_) (void)hipSetDevice(prev_); }
    bool ok() const { return dev_ >= 0; }
    // p is memory of this call's device: a host pointer or another device's would fault the kernel or cross the fabric unseen
    bool owns(const void *p) const {
        if (!p) return false;
        hipPointerAttribute_t a;
        if (hipPointerGetAttributes(&a, p) != hipSuccess) { (void)hipGetLastError(); return false; }
        return (a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged) && a.device == dev_;
    }
    template <class... P> bool own(P... p) const { return (owns(p) && ...); }

private:
    int dev_ = -1, prev_ = -1;
};

// A launch by its own status: the runtime's last error may be another call's, from before, and is neither reported nor cleared.
template <class... P> inline bool serve_launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, P... args) {
    void *ptrs[] = {(void *)&args...};
    if (hipLaunchKernel((const void *)kernel, grid, block, ptrs, lds, st) == hipSuccess) return true;
    (void)hipGetLastError();
    return false;
}

}  // namespace wmi
