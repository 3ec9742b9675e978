// Shared by the kernels of the quantised head: element types, MXFP4 rows, the error word.
#pragma once
#include <atomic>

#include "dsx_common.cuh"

namespace dsx {


// ------------------------------------------------------------ element types
template <int DT> struct Elem;
template <> struct Elem<DSX_F32> { using T = float; };
template <> struct Elem<DSX_BF16> { using T = __nv_bfloat16; };
template <> struct Elem<DSX_F16> { using T = __half; };

__host__ __device__ inline bool dtype_ok(int dt) { return dt == DSX_F32 || dt == DSX_BF16 || dt == DSX_F16; }
__host__ __device__ inline int dtype_size(int dt) { return dt == DSX_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
// The one rounding of a result to its type (nearest even).
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// Two values as one 32-bit word of a 16-bit type, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// SM count of the current device, looked up once per device.
inline int head_sm_count(int* sms) {
    constexpr int kMaxDevices = 64;
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    DSX_CUDA(cudaGetDevice(&dev));
    DSX_REQUIRE(dev >= 0 && dev < kMaxDevices, "device index %d out of range", dev);
    int n = known[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        DSX_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        known[dev].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return DSX_OK;
}

// -------------------------------------------------------------- MXFP4 values
// 2^(e - 127); e = 0 is the subnormal 2^-127, e = 255 is NaN (the E8M0 encoding).
__device__ __forceinline__ float e8m0_value(uint32_t e) {
    return e == 255u ? __uint_as_float(0x7FC00000u) : (e == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(e << 23));
}
// Value of the E2M1 code in the low four bits of n, times 2^-126: two exponent bits and the mantissa bit sit where an f32 has
// its lowest exponent bits and its highest mantissa bit (code 1 is the f32 subnormal 2^-127, as it is E2M1's own subnormal 0.5).
__device__ __forceinline__ float e2m1_scaled(uint32_t n) { return __uint_as_float(((n & 7u) << 22) | ((n & 8u) << 28)); }
// * 2^126, exact; adding +0 turns code 8 (minus zero) into plain zero, as the CPU quantiser's integer table has it, so that the sign of a
// zero residual -- and with it the code of the next term -- is the same there
__device__ __forceinline__ float e2m1_to_f32(uint32_t n) { return __fmaf_rn(e2m1_scaled(n), 8.507059173023462e37f, 0.0f); }

}  // namespace dsx
