// What the C-ABI entry points of the step operators share (step_api.cpp, step_mix_api.cpp): errors, and the checks of pointers and
// streams.
#pragma once
#include "step_launch.h"

#include <hip/hip_runtime.h>

#include <stdexcept>
#include <string>

namespace qkv {

void set_error(const char * msg); // kv_api.cpp: mk_last_error's message

namespace { // (each source its own)

template <class R, class F> R guarded(F f) {
    try {
        return f();
    } catch (const std::exception & e) {
        set_error(e.what());
    } catch (...) {
        set_error("unknown exception");
    }
    return -1;
}

[[noreturn]] void bad(const std::string & msg) { throw std::runtime_error(msg); }

void ck(hipError_t e, const char * what) {
    if (e == hipSuccess) return;
    (void) hipGetLastError(); // (reported here, not by a later call)
    bad(std::string(what) + ": " + hipGetErrorString(e));
}

// the stream is of the current device, and every buffer is memory of it (a host address or another device's would fault the GPU)
struct Device {
    int dev = -1;
    explicit Device(void * stream) {
        ck(hipGetDevice(&dev), "hipGetDevice");
        if (!stream || stream == hipStreamLegacy || stream == hipStreamPerThread) return; // (of the current device)
        hipDevice_t of = -1;
        ck(hipStreamGetDevice(static_cast<hipStream_t>(stream), &of), "stream");
        if (of != dev) bad("stream is of device " + std::to_string(of) + ", the current device is " + std::to_string(dev));
    }
    void holds(const void * p, const char * name) const {
        if (!p) return;
        hipPointerAttribute_t at{};
        const hipError_t e = hipPointerGetAttributes(&at, p);
        if (e != hipSuccess) (void) hipGetLastError(); // (reported here, not by a later call)
        if (e != hipSuccess || (at.type != hipMemoryTypeDevice && at.type != hipMemoryTypeManaged)) bad(std::string(name) + " is not device memory");
        if (at.device != dev)
            bad(std::string(name) + " is memory of device " + std::to_string(at.device) + ", the current device is " + std::to_string(dev));
    }
};

void need(const void * p, const char * name) {
    if (!p) bad(std::string("null ") + name + " pointer");
}
void aligned(const void * p, unsigned to, const char * name) {
    if ((uintptr_t) p % to) bad(std::string(name) + " is not aligned to " + std::to_string(to) + " bytes");
}
unsigned size_of(int dtype) {
    if (dtype < DT_F32 || dtype > DT_BF16) bad("dtype: 0 fp32, 1 fp16, 2 bf16");
    return dtype == DT_F32 ? 4 : 2;
}

} // namespace
} // namespace qkv
