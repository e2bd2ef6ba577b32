// Host-side helpers shared by the translation units of the C ABI.
#pragma once

#include <cuda_runtime.h>
#include <stdlib.h>

#include "../../include/ue5m3_fp4.h"

namespace ue5m3 {

// Number of SMs of the current device (cached per device ordinal).
int sm_count();

// cudaGetLastError() -> status code; records the error text for
// ue5m3_last_cuda_error().
int check_launch();
int record_cuda_error(cudaError_t error);
void record_error_text(const char* text);

// Dynamic shared memory above 48 KiB has to be asked for once per kernel and device.
template <auto kKernel>
cudaError_t allow_shared(int bytes) {
    static bool done[64] = {};
    int device = 0;
    cudaError_t error = cudaGetDevice(&device);
    if (error != cudaSuccess || (device < 64 && done[device])) return error;
    error = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (error == cudaSuccess && device < 64) done[device] = true;
    return error;
}

}  // namespace ue5m3
