/* makes a device current for the calling thread while the guard lives */
#ifndef DEVICE_GUARD_H
#define DEVICE_GUARD_H

#include <cuda_runtime.h>

struct DeviceGuard {
    int before = -1;
    bool ok = false;
    explicit DeviceGuard(int device)
    {
        int now = -1;
        if (device < 0)
            return;
        if (cudaGetDevice(&now) != cudaSuccess || (now != device && cudaSetDevice(device) != cudaSuccess)) {
            cudaGetLastError();     /* reported here, and not left for a later call to find */
            return;
        }
        if (now != device)
            before = now;
        ok = true;
    }
    ~DeviceGuard()
    {
        if (before >= 0)
            cudaSetDevice(before);
    }
};

#endif
