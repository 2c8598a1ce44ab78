// What the operators on scores and rows share: value types, the device and stream of a call, launches.
#pragma once

#include "operators.h"

#include <hip/hip_runtime.h>

#include <cstdint>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>

namespace cbamd {
namespace op {

inline void Check(hipError_t e, const char* what) {
    if (e != hipSuccess) {
        throw TModelError(std::string("HIP error in ") + what + ": " + hipGetErrorString(e));
    }
}
#define OP_HIP_CHECK(expr) ::cbamd::op::Check((expr), #expr)

// The device that a call's output is on is the thread's current one for as long as this lives. The operators have no
// handle that knows a device, so the output's address tells it; a stream of another device is refused.
class TCallDevice {
public:
    // (hipStreamLegacy is another name of the default stream, which hipStreamGetDevice takes for an address)
    TCallDevice(const void* output, void* stream)
        : Stream(stream != static_cast<void*>(hipStreamLegacy) ? static_cast<hipStream_t>(stream) : nullptr)
    {
        hipPointerAttribute_t attributes;
        if (hipPointerGetAttributes(&attributes, output) != hipSuccess || attributes.type == hipMemoryTypeUnregistered) {
            (void)hipGetLastError();  // what this call left is no later one's
            throw TModelError("the output is not in memory that a GPU can write");
        }
        if (Stream != nullptr) {
            hipDevice_t device = 0;
            OP_HIP_CHECK(hipStreamGetDevice(Stream, &device));
            CBAMD_ENSURE(device == attributes.device, "the stream and the output are on different devices");
        }
        Device = attributes.device;
        OP_HIP_CHECK(hipGetDevice(&Previous));
        if (Previous != Device) {
            OP_HIP_CHECK(hipSetDevice(Device));
            Changed = true;
        }
    }
    ~TCallDevice() {
        if (Changed) {
            (void)hipSetDevice(Previous);
        }
    }
    TCallDevice(const TCallDevice&) = delete;
    TCallDevice& operator=(const TCallDevice&) = delete;

    // (the launch's own status: hipGetLastError would also hand over what another library's call left behind)
    template <typename... TParams, typename... TArgs>
    void Launch(void (*kernel)(TParams...), size_t groups, uint32_t threads, size_t ldsBytes, TArgs&&... args) const {
        std::tuple<TParams...> held(std::forward<TArgs>(args)...);
        LaunchHeld(reinterpret_cast<const void*>(kernel), groups, threads, ldsBytes, held,
                   std::index_sequence_for<TParams...>());
    }

    // A kernel that uses more than 64 KB of LDS has to be told so, for each device; the largest size so far is remembered.
    // `bytes`: the dynamic part (the kernels here have under 1 KB beside it)
    void AllowLds(const void* kernel, size_t bytes) const {
        if (bytes <= 63 * 1024) {
            return;
        }
        static std::mutex lock;
        static std::map<std::pair<int, const void*>, size_t> allowed;
        std::lock_guard<std::mutex> guard(lock);
        size_t& most = allowed[{Device, kernel}];
        if (most < bytes) {
            OP_HIP_CHECK(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
            most = bytes;
        }
    }

private:
    template <typename TTuple, size_t... I>
    void LaunchHeld(const void* kernel, size_t groups, uint32_t threads, size_t ldsBytes, TTuple& held,
                    std::index_sequence<I...>) const {
        void* args[] = {static_cast<void*>(&std::get<I>(held))...};
        OP_HIP_CHECK(hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(groups)), dim3(threads), args, ldsBytes, Stream));
    }

    hipStream_t Stream = nullptr;
    int Device = 0;
    int Previous = 0;
    bool Changed = false;
};

// Sums, softmax statistics and everything between a load and a store are in 32 bits, in 64 for 64-bit values
template <typename T>
struct TAccumulator {
    using Type = float;
};
template <>
struct TAccumulator<double> {
    using Type = double;
};
template <typename T>
using TAcc = typename TAccumulator<T>::Type;

// f(T()) for the C++ type of a value type
template <typename F>
void WithType(int valueType, F&& f) {
    switch (valueType) {
        case CBHIP_FLOAT64: return f(double());
        case CBHIP_FLOAT32: return f(float());
        case CBHIP_FLOAT16: return f(_Float16());
        case CBHIP_BFLOAT16: return f(__bf16());
    }
    CBAMD_ENSURE(false, "unknown value type " + std::to_string(valueType));
}

inline size_t ValueSize(int valueType) {
    CBAMD_ENSURE(valueType >= CBHIP_FLOAT64 && valueType <= CBHIP_BFLOAT16, "unknown value type " + std::to_string(valueType));
    return valueType == CBHIP_FLOAT64 ? 8 : valueType == CBHIP_FLOAT32 ? 4 : 2;
}

// A matrix of `rows` rows of `width` values, `stride` values from row to row: what every operand is asked
inline void CheckMatrix(const char* name, const void* data, size_t rows, size_t width, size_t stride, size_t valueSize) {
    CBAMD_ENSURE(data != nullptr, std::string(name) + " pointer is null");
    CBAMD_ENSURE(rows <= 1 || stride >= width, std::string(name) + ": a stride of " + std::to_string(stride) +
                                                   " values is shorter than a row of " + std::to_string(width));
    CBAMD_ENSURE(reinterpret_cast<uintptr_t>(data) % valueSize == 0, std::string(name) + " pointer is not a multiple of the value size");
    CBAMD_ENSURE(rows <= 1 || stride <= (size_t(1) << 60) / valueSize / rows, std::string(name) + " is too large");
}

// What lanes of a wave hand each other through LDS: a wave's LDS operations are done in order, so that there is nothing to
// wait for; the fences keep the compiler from moving them across (they cost no instruction)
__device__ __forceinline__ void WaveHandover() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// N values in a row, at any alignment of what they are loaded from or stored to, whose type the pointer says (words of a
// row of 16-bit values are at multiples of 2): one wide load or store where N values make one (the hardware's unaligned
// mode takes any address)
template <typename T, int N>
struct TValues {
    T V[N];
    template <typename TFrom>
    __device__ __forceinline__ static TValues Load(const TFrom* at) {
        TValues r;
        __builtin_memcpy(&r, at, sizeof(r));
        return r;
    }
    template <typename TTo>
    __device__ __forceinline__ void Store(TTo* at) const {
        __builtin_memcpy(at, this, sizeof(*this));
    }
};

// The same for the `n` values that are left of a row, where those are fewer
template <typename T, int N>
__device__ __forceinline__ TValues<T, N> LoadUpTo(const T* at, size_t n) {
    if (n >= N) {
        return TValues<T, N>::Load(at);
    }
    TValues<T, N> v{};
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (static_cast<size_t>(i) < n) {
            v.V[i] = at[i];
        }
    }
    return v;
}
template <typename T, int N>
__device__ __forceinline__ void StoreUpTo(const TValues<T, N>& v, T* at, size_t n) {
    if (n >= N) {
        v.Store(at);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (static_cast<size_t>(i) < n) {
            at[i] = v.V[i];
        }
    }
}

}  // namespace op
}  // namespace cbamd
