// vtx_host.cuh — host helpers shared by the library's translation units:
// per-device state, size arithmetic and the programmatic-dependent-launch
// wrapper.  Nothing here allocates, synchronises or aborts.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <cstddef>
#include <cstdint>
#include <utility>

#include "../../include/vtx_fa.h"

namespace vtx {

constexpr int kMaxDevices = 64;

struct DeviceState {
    int ok = 0;
    int sms = 148;
    int *err = nullptr;       // device error word of this device
};

// State of the current device, set up on its first use; VTX_ERR_NO_DEVICE
// when it is not an sm_100 device.  Defined in vtx_fa.cu.
int ensure_device(DeviceState **out);
// cuTensorMapEncodeTiled, looked up with the first device (NULL before, or
// when the driver lacks it).  Defined in vtx_fa.cu.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline int elem_size(int t) { return t == VTX_TYPE_F32 ? 4 : 2; }
inline int row_bytes(int t, int64_t d) { return t == VTX_TYPE_Q8_0 ? (int)(d / 32 * 34) : (int)(d * elem_size(t)); }

// Every kernel is launched with programmatic stream serialisation (PDL): it
// may be scheduled while the previous kernel on the stream drains, and waits
// for it in-kernel (grid_dep_wait) before touching global memory.
template <typename... KArgs, typename... Args>
int launch_pdl(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...) == cudaSuccess ? VTX_OK : VTX_ERR_CUDA;
}

}  // namespace vtx
