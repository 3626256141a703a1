// What the operators' host sides share: checks of arguments, the current device, launch errors.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "../cuda/capi_cuda.h"
#include "capi_train.h"

namespace stdml::collective::cuda
{
void set_last_error(const std::string &msg);  // capi_cuda.cpp
}

namespace stdml::collective::train
{
inline void require(bool ok, const char *what)
{
    if (!ok) { throw std::invalid_argument(what); }
}

inline void cuda_ok(cudaError_t e, const char *what)
{
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
    }
}

// The GPU of a call is current while it launches, and the caller's again afterwards.
class CurrentDevice
{
  public:
    explicit CurrentDevice(int device)
    {
        cuda_ok(cudaGetDevice(&before_), "cudaGetDevice");
        if (before_ != device) { cuda_ok(cudaSetDevice(device), "cudaSetDevice"); }
        moved_ = before_ != device;
    }
    ~CurrentDevice()
    {
        if (moved_) { (void)cudaSetDevice(before_); }
    }
    CurrentDevice(const CurrentDevice &) = delete;

  private:
    int before_ = 0;
    bool moved_ = false;
};

// Nothing may unwind through the C boundary.
template <typename F>
int entry(int device, F f)
{
    try {
        const CurrentDevice on(device);
        f();
        cuda_ok(cudaGetLastError(), "kernel launch");
        return STDMLC_OK;
    } catch (const std::invalid_argument &e) {
        cuda::set_last_error(e.what());
        return STDMLC_ERR_ARGS;
    } catch (const std::exception &e) {
        cuda::set_last_error(e.what());
        return STDMLC_ERR_RUNTIME;
    } catch (...) {
        cuda::set_last_error("unknown C++ exception");
        return STDMLC_ERR_RUNTIME;
    }
}

// The same for a number of bytes: -1 where there is none.
template <typename F>
long long bytes_entry(F f)
{
    try {
        return f();
    } catch (const std::exception &e) {
        cuda::set_last_error(e.what());
    } catch (...) {
        cuda::set_last_error("unknown C++ exception");
    }
    return -1;
}

inline int sm_count()
{
    int dev = 0, n = 0;
    cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
    cuda_ok(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "SM count");
    return n;
}

inline int element_size(int dt) { return dt == 10 ? 4 : 2; }
inline bool float_type(int dt) { return dt >= 8 && dt <= 10; }
}  // namespace stdml::collective::train
