// The frame of an operator entry that works on the caller's device buffers: makes the buffers' device current for the
// call and the caller's again afterwards, and turns CUDA errors into a reason (these entries never end the process).
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdio.h>
#include <string.h>

namespace ntcb {

inline void set_why(char* why, size_t cap, const char* msg) {
    if (why && cap) { strncpy(why, msg, cap - 1); why[cap - 1] = 0; }
}

// SM count of a device, 0 when it cannot be asked for (device_cache.cu keeps it per device, without ending the process).
int device_sm_count_or_zero(int device);

struct DeviceScope {
    int before = -1, device = -1, sms = 0;
    bool ok = false;
    // device < 0: the current one. A CUDA error that is already pending is reported and left pending: the call could not
    // tell its own launch errors from it.
    DeviceScope(int want, char* why, size_t cap) {
        cudaError_t e = cudaPeekAtLastError();
        if (e != cudaSuccess) { fail("a CUDA error was pending before the call", e, why, cap); return; }
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && want >= 0 && want != before) e = cudaSetDevice(want);
        device = want >= 0 ? want : before;
        if (e == cudaSuccess && (sms = device_sm_count_or_zero(device)) == 0) e = cudaErrorInvalidDevice;
        if (e != cudaSuccess) { cudaGetLastError(); fail("no usable CUDA device", e, why, cap); return; }
        ok = true;
    }
    ~DeviceScope() { if (before >= 0 && device != before) cudaSetDevice(before); }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    int launched(cudaError_t e, char* why, size_t cap) {
        if (e == cudaSuccess) return 1;
        cudaGetLastError();
        fail("a kernel launch failed", e, why, cap);
        return 0;
    }
    static void fail(const char* where, cudaError_t e, char* why, size_t cap) {
        if (why && cap) snprintf(why, cap, "%s: %s", where, cudaGetErrorString(e));
    }
};

}  // namespace ntcb
