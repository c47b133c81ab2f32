// The context's device for the length of a call; the caller's is set again behind it.
#pragma once
#include <cuda_runtime_api.h>

namespace mpq {

class OnDevice {
public:
    explicit OnDevice(int device)
    {
        if ((error = cudaGetDevice(&before_)) == cudaSuccess && before_ != device && (error = cudaSetDevice(device)) == cudaSuccess) moved_ = true;
    }
    ~OnDevice() { if (moved_) cudaSetDevice(before_); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
    cudaError_t error;

private:
    int before_ = 0;
    bool moved_ = false;
};

}  // namespace mpq
