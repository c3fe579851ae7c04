// Host-side helpers shared by the files that implement the C ABI: status codes with a message,
// the device scope, device memory, and the ordering of calls that share a workspace.
#pragma once
#include "../../include/ek_hip.h"
#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <exception>
#include <new>

namespace ek {

void set_last_error(const char *msg);

__attribute__((format(printf, 2, 3))) inline ek_status fail(ek_status st, const char *fmt, ...)
{
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    set_last_error(buf);
    return st;
}

inline ek_status hip_fail(hipError_t e, const char *what)
{
    (void)hipGetLastError();   // clear the sticky error
    return fail(e == hipErrorOutOfMemory ? EK_OOM : EK_HIP_ERROR, "%s: %s", what, hipGetErrorString(e));
}

#define EK_HIP(call)                                                  \
    do {                                                              \
        hipError_t _e = (call);                                       \
        if (_e != hipSuccess) return ek::hip_fail(_e, #call);         \
    } while (0)

#define EK_TRY(call)                                                  \
    do {                                                              \
        ek_status _s = (call);                                        \
        if (_s != EK_OK) return _s;                                   \
    } while (0)

#define EK_GUARDED(...)                                               \
    try {                                                             \
        __VA_ARGS__                                                   \
    } catch (const std::bad_alloc &) {                                \
        return ek::fail(EK_OOM, "host allocation failed");            \
    } catch (const std::exception &ex) {                              \
        return ek::fail(EK_INTERNAL, "exception: %s", ex.what());     \
    } catch (...) {                                                   \
        return ek::fail(EK_INTERNAL, "unknown exception");            \
    }

// Makes `dev` current for the scope and restores the caller's device.
struct DeviceGuard {
    int prev = -1;
    bool ok = false;
    explicit DeviceGuard(int dev)
    {
        if (hipGetDevice(&prev) != hipSuccess) { (void)hipGetLastError(); prev = -1; }
        if (prev == dev) { ok = true; prev = -1; return; }
        ok = hipSetDevice(dev) == hipSuccess;
        if (!ok) (void)hipGetLastError();
    }
    ~DeviceGuard()
    {
        if (prev >= 0 && ok) (void)hipSetDevice(prev);
    }
};

inline ek_status dev_alloc(void **p, size_t bytes, const char *what)
{
    hipError_t e = hipMalloc(p, bytes ? bytes : 16);
    if (e != hipSuccess) {
        *p = nullptr;
        (void)hipGetLastError();
        return fail(e == hipErrorOutOfMemory ? EK_OOM : EK_HIP_ERROR, "hipMalloc(%s, %zu bytes): %s",
                    what, bytes, hipGetErrorString(e));
    }
    return EK_OK;
}

inline bool stream_capturing(hipStream_t s)
{
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &cs) != hipSuccess) { (void)hipGetLastError(); return false; }
    return cs != hipStreamCaptureStatusNone;
}

// One use of a workspace on stream s; the caller holds the lock that guards it for the scope.
// begin(): the stream waits (on the device) for the last enqueue-only call that used the
// workspace.  At the end of the scope the stream's position is recorded as that call's end,
// unless synced() says the host has waited for the stream, after which nothing is pending.
// A stream under capture by the caller is left alone both ways (a captured wait on an event
// recorded outside the capture is not allowed): replays of such a graph use the workspace like
// the call they record, and ordering them against other calls on the layer is the caller's part.
struct WorkspaceUse {
    hipEvent_t ev;
    bool *busy;
    hipStream_t s;
    bool capturing = false, host_synced = false;
    WorkspaceUse(hipEvent_t event, bool *busy_flag, hipStream_t stream) : ev(event), busy(busy_flag), s(stream) {}
    ek_status begin()
    {
        capturing = stream_capturing(s);
        if (!capturing && *busy) EK_HIP(hipStreamWaitEvent(s, ev, 0));
        return EK_OK;
    }
    void device_idle() { *busy = false; }          // after a hipDeviceSynchronize
    void synced() { host_synced = true; }          // after a hipStreamSynchronize(s) that followed begin()
    ~WorkspaceUse()
    {
        if (capturing) return;
        if (host_synced) { *busy = false; return; }
        if (hipEventRecord(ev, s) == hipSuccess) *busy = true;
        else (void)hipGetLastError();
    }
};

}  // namespace ek
