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

// Programmatic launches: the next kernel of a call starts while this one ends, and waits for it
// where it first reads what this one writes.
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_launcher() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

// Clusters of `size` CTAs that the current device holds at a time (0: none, or an error), asked for
// once per kernel, device and size.
template <auto kKernel>
int resident_clusters(int size, int threads, int shared) {
    static int known[64][9] = {};
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device >= 64 || size > 8) return 0;
    if (known[device][size] == 0) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(size);
        config.blockDim = dim3(threads);
        config.dynamicSmemBytes = shared;
        cudaLaunchAttribute attribute;
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = size;
        attribute.val.clusterDim.y = 1;
        attribute.val.clusterDim.z = 1;
        config.attrs = &attribute;
        config.numAttrs = 1;
        int count = 0;
        if (cudaOccupancyMaxActiveClusters(&count, kKernel, &config) != cudaSuccess) {
            cudaGetLastError();
            count = 0;
        }
        known[device][size] = count > 0 ? count : -1;
    }
    return known[device][size] > 0 ? known[device][size] : 0;
}

}  // namespace ue5m3
