// What the entry points of the optimiser and of the table lookups share.
#pragma once
#include "splat_internal.h"

#include "../../include/trips_optim.h"

namespace trips
{
// Work goes to the context's device; the caller's current device is put back.
struct DeviceScope
{
    int previous = -1;
    hipError_t error;
    explicit DeviceScope(int device)
    {
        int now = -1;
        error   = hipGetDevice(&now);
        if (error != hipSuccess || now == device) return;
        error = hipSetDevice(device);
        if (error == hipSuccess) previous = now;
    }
    ~DeviceScope()
    {
        if (previous >= 0) (void)hipSetDevice(previous);
    }
    DeviceScope(const DeviceScope&)            = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;
};

inline int hip_error(hipError_t e, const char* what) { return set_error(TRIPS_ERR_HIP, "%s: %s", what, hipGetErrorString(e)); }
inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }
inline bool dtype_ok(int d) { return d == TRIPS_DTYPE_F32 || d == TRIPS_DTYPE_BF16 || d == TRIPS_DTYPE_F16; }
inline int dtype_bytes(int d) { return d == TRIPS_DTYPE_F32 ? 4 : 2; }
inline Profiler* profiler(TripsCtx* ctx) { return ctx->prof.enabled ? &ctx->prof : nullptr; }

// The element types: how they are held, and their way to and from float (rounded to nearest, ties to even).
template <int DTYPE>
struct Element;
template <>
struct Element<TRIPS_DTYPE_F32>
{
    using type = float;
    static __device__ __forceinline__ float to_float(float x) { return x; }
    static __device__ __forceinline__ float from_float(float x) { return x; }
};
template <>
struct Element<TRIPS_DTYPE_BF16>
{
    using type = unsigned short;
    static __device__ __forceinline__ float to_float(unsigned short x) { return __uint_as_float((unsigned)x << 16); }
    static __device__ __forceinline__ unsigned short from_float(float x) { return __builtin_bit_cast(unsigned short, (__bf16)x); }
};
template <>
struct Element<TRIPS_DTYPE_F16>
{
    using type = unsigned short;
    static __device__ __forceinline__ float to_float(unsigned short x) { return (float)__builtin_bit_cast(_Float16, x); }
    static __device__ __forceinline__ unsigned short from_float(float x) { return __builtin_bit_cast(unsigned short, (_Float16)x); }
};

// Pointers that a kernel finds in memory: said to be global (the compiler would take them for any kind), or to a table that no
// kernel writes while this one runs (read by scalar loads).
template <typename T>
using Global = __attribute__((address_space(1))) T*;
template <typename T>
using Constant = const __attribute__((address_space(4))) T*;
template <typename T>
__device__ __forceinline__ Global<T> global(T* p)
{
    return (Global<T>)p;
}

// N elements side by side, at any address that their type allows (global memory takes wide accesses there too).
template <typename T, int N>
struct Pack
{
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
}  // namespace trips
