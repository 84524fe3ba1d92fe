// Host helpers of the serving ops: argument checks, the device guard, and the
// C entry's error boundary.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <exception>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "kernels.h"
#include "kv4.cuh"
#include "needle_engine.h"

namespace nd {

void set_error(const std::string& msg);

// Makes `device` current for a scope.
struct OnDevice {
    int prev = -1;
    OnDevice(int device, const char* what) {
        cudaError_t e = cudaGetDevice(&prev);
        if (e == cudaSuccess && prev != device) e = cudaSetDevice(device);
        else if (e == cudaSuccess) prev = -1;
        if (e != cudaSuccess) {
            prev = -1;
            cudaGetLastError();
            throw std::runtime_error(std::string(what) + ": device " + std::to_string(device) + ": " + cudaGetErrorString(e));
        }
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

// Runs a C entry's body: 0, or -1 with its message kept for nd_last_error.
template <typename F>
int op_call(F&& f) {
    try {
        f();
        return 0;
    } catch (std::exception& e) {
        try {
            set_error(e.what());
        } catch (...) {
        }
        return -1;
    } catch (...) {
        return -1;
    }
}

// A launch's error as an exception; counts the launches otherwise.
inline void op_launched(const char* what, int kernels = 1) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
    add_launches(kernels);
}

// Lets a kernel have `bytes` of shared memory, once a device: the call costs
// a microsecond.
template <auto Kernel>
void allow_smem(int bytes, const char* what) {
    static std::atomic<unsigned long long> done{0};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const unsigned long long bit = device < 64 ? 1ull << device : 0;
    if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
        e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess) done.fetch_or(bit);
    }
    if (e != cudaSuccess) throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
}

Kv4Args kv4_args(const nd_kv4* kv, const char* what);
// 16-byte loads and stores of eight elements are aligned for these rows.
bool kv4_vec(int type, const void* p, long long row, long long head);
void kv4_check_rows(const char* what, int type, const void* p, long long row, long long head);
void kv4_check_out(const char* what, int type, const void* p, long long row, long long head, int rows, int heads, int d);

}  // namespace nd
