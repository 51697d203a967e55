// rt_internal.h — runtime helpers shared by the HIP translation units of
// libwelvet_hip (defined in runtime.hip). HIP-only: includes hip_runtime.h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "wv_internal.h"

namespace wv {

// Sets the calling thread's wv_last_error() text and returns `code`.
int rt_fail(int code, const char* fmt, ...);
// Maps a HIP error to WV_E_OOM / WV_E_HIP with context `what`.
int rt_hip_fail(hipError_t e, const char* what);
// Initialises device 0 unless wv_init chose one; makes it current.
int rt_ensure_init();
// Copies the device view of blob `h`; false if the handle is unknown.
bool rt_lookup(uint64_t h, DevBlob& out);
// The device wv_init selected (-1 before any init).
int rt_current_device();
// `stream`, or the library's own stream of `device` for NULL.
hipStream_t rt_stream(void* stream, int device);
// Whether `s` is being captured into a HIP graph.
bool rt_capturing(hipStream_t s);

// A slot of the current device's per-call scratch (CallScratch, runtime.hip):
// held from get() until this object goes, which has to be after the call's
// last launch. Not for a stream under capture.
class RtScratch {
public:
    RtScratch() = default;
    RtScratch(const RtScratch&) = delete;
    RtScratch& operator=(const RtScratch&) = delete;
    ~RtScratch();
    int get(size_t floats, hipStream_t s, const char* what);
    float* f() const;

private:
    void* impl_ = nullptr;
};

}  // namespace wv
