// What the parts of the torch library share (extension.cpp, block_extension.cpp): host code only, torch's stable ABI.
#pragma once

#include <torch/csrc/stable/accelerator.h>
#include <torch/csrc/stable/tensor.h>

#include <hip/hip_runtime_api.h>

#include <cstdint>

inline bool is_aligned(const void* p, uintptr_t bytes) {
    return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

inline hipStream_t current_stream(int32_t device_index) {
    void* raw_stream = nullptr;
    TORCH_ERROR_CODE_CHECK(aoti_torch_get_current_cuda_stream(device_index, &raw_stream));
    return static_cast<hipStream_t>(raw_stream);
}

inline void check_launch(bool launched, const char* what) {
    STD_TORCH_CHECK(launched, "Unsupported config");
    const hipError_t err = hipGetLastError();
    STD_TORCH_CHECK(err == hipSuccess, what, " kernel launch failed: ", hipGetErrorString(err));
}
