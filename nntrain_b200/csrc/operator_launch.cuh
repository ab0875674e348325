// Host plumbing shared by the training operators (list norm, RMS norm, token
// table): the caller's device is put back when an entry point returns, every
// launch answers with its own status, and dependent kernels are launched so that
// their prologue overlaps the end of the kernel in front of them.
#pragma once

#include "common.cuh"

namespace ngb {

// A failed runtime call also stays behind as the thread's last error, where the
// next check of any library in the process takes it for its own.  Here the entry
// point's status tells it, so it is taken away.
inline cudaError_t reported(cudaError_t status) {
    if (status != cudaSuccess) cudaGetLastError();
    return status;
}

// Selects `device` for the calling thread and selects the previous one again
// at the end of the scope.
class DeviceScope {
public:
    explicit DeviceScope(int device) : device_(device) {
        if (reported(cudaGetDevice(&previous_)) != cudaSuccess) previous_ = -1;
        status_ = select_device(device);
    }
    ~DeviceScope() {
        if (previous_ >= 0 && previous_ != device_ && status_ == static_cast<int>(cudaSuccess)) select_device(previous_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
    int status() const { return status_; }

private:
    int device_, previous_ = -1, status_ = 0;
};

inline bool aligned_for(const void* p, std::uintptr_t bytes) {
    return (reinterpret_cast<std::uintptr_t>(p) & (bytes - 1)) == 0;
}

#ifdef __CUDACC__

// The status is this launch's own: peeking at the last error would also find one
// that an earlier call on this thread left there.
template <typename... Parameters, typename... Arguments>
cudaError_t launch_with(cudaLaunchAttribute* attributes, int count, void (*kernel)(Parameters...), dim3 grid, int threads,
                        size_t shared, cudaStream_t stream, Arguments... arguments) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    config.attrs = attributes;
    config.numAttrs = count;
    return reported(cudaLaunchKernelEx(&config, kernel, static_cast<Parameters>(arguments)...));
}

template <typename... Parameters, typename... Arguments>
cudaError_t launch(void (*kernel)(Parameters...), dim3 grid, int threads, size_t shared, cudaStream_t stream,
                   Arguments... arguments) {
    return launch_with(nullptr, 0, kernel, grid, threads, shared, stream, arguments...);
}

// Launches `kernel` behind the kernel in front of it on `stream` with
// programmatic serialization: its CTAs may be resident before that kernel has
// ended, and wait_for_previous() in it returns once all of that kernel's
// writes are visible.  Every kernel launched this way calls it before its
// first read of anything another kernel writes, and before its first write.
template <typename... Parameters, typename... Arguments>
cudaError_t launch_dependent(void (*kernel)(Parameters...), int grid, int threads, size_t shared, cudaStream_t stream,
                             Arguments... arguments) {
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    return launch_with(&attribute, 1, kernel, dim3(static_cast<unsigned>(grid)), threads, shared, stream, arguments...);
}

__device__ __forceinline__ void wait_for_previous() { cudaGridDependencySynchronize(); }
__device__ __forceinline__ void let_next_start() { cudaTriggerProgrammaticLaunchCompletion(); }

// Two fp32 values -> two bf16 (round to nearest even, NaN -> 0x7fff), the
// first in the low half.
__device__ __forceinline__ unsigned pack_bf16(float low, float high) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(low, high);
    return *reinterpret_cast<const unsigned*>(&v);
}
__device__ __forceinline__ float bf16_low(unsigned word) { return __uint_as_float(word << 16); }
__device__ __forceinline__ float bf16_high(unsigned word) { return __uint_as_float(word & 0xffff0000u); }
__device__ __forceinline__ float bf16_value(unsigned short bits) {
    return __uint_as_float(static_cast<unsigned>(bits) << 16);
}
__device__ __forceinline__ unsigned short bf16_bits(float value) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(value));
}

#endif  // __CUDACC__

}  // namespace ngb
