// Shared by the kernels of the quantised head: element types, pairs of f32, MXFP4 values.
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

// Two f32 in one register pair.
__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

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
// The codes in nibble k of either half of x as two f16 values: the two exponent bits and the mantissa bit of a code sit where an f16 has its
// lowest exponent bits and its highest mantissa bit (code 1 is an f16 subnormal there, as it is E2M1's own), so what is left is a factor of 2^14.
// Four integer instructions a pair.  (The hardware's decoder, cvt.rn.f16x2.e2m1x2, is two instructions shorter.  Twice it gave other values than
// the codes stand for in a kernel although it is right in isolation (CUDA 12.9, sm_100a): zeros in a build of the dequantiser to f32, wrong residuals in
// the layer's quantiser of activations.  The cause is not known.  The library uses it in the decode kernels, the f16-operand kernels
// and, behind an exclusive-or, that quantiser, whose results the tests hold against the CPU's; the encoder's codes (mxfp4_rows.cu) are compared bit for bit.)
template <int K>
__device__ __forceinline__ float2 e2m1_pair(uint32_t x) {
    const uint32_t mag = K == 0 ? x << 9 : (K == 1 ? x << 5 : (K == 2 ? x << 1 : x >> 3));
    const uint32_t sign = K == 0 ? x << 12 : (K == 1 ? x << 8 : (K == 2 ? x << 4 : x));
    const uint32_t h = (mag & 0x0E000E00u) | (sign & 0x80008000u);
    return __half22float2(__hmul2(*reinterpret_cast<const __half2*>(&h), __half2half2(__ushort_as_half((unsigned short)0x7400))));   // * 2^14
}
// The values of eight codes (element i in nibble i), and of four in the low half of w.  Exact.
__device__ __forceinline__ void e2m1_values(uint32_t w, float (&d)[8]) {
    const float2 a = e2m1_pair<0>(w), b = e2m1_pair<1>(w), c = e2m1_pair<2>(w), e = e2m1_pair<3>(w);
    d[0] = a.x; d[4] = a.y; d[1] = b.x; d[5] = b.y; d[2] = c.x; d[6] = c.y; d[3] = e.x; d[7] = e.y;
}
__device__ __forceinline__ void e2m1_values(uint32_t w, float (&d)[4]) {
    const uint32_t x = __byte_perm(w, 0u, 0x4140);   // byte 0 to the low half, byte 1 to the high one
    const float2 a = e2m1_pair<0>(x), b = e2m1_pair<1>(x);
    d[0] = a.x; d[2] = a.y; d[1] = b.x; d[3] = b.y;
}

}  // namespace dsx
