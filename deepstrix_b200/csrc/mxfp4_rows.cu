// Rows of f32 / bf16 / f16 values as sums of MXFP4 terms, and back.
//
// Reference counterparts (paths relative to the deepstrix repository): the FP4 fake-quantiser of its CPU model
// (scripts/v41_oracle/kernel.py:129-147) and the byte layout its loader reads (crates/v4flash-core/src/hf_v41.rs:1150-1233).
//
// A term of a block of 32 values r:  e = E - 2 (+ 1 when m > 1.5) for the largest magnitude m * 2^E, kept in 1..253 -- that is
// 127 + ceil(log2(max |r| / 6)), the smallest power of two that brings the block into E2M1's range -- code = r / 2^(e-127) rounded to
// the nearest E2M1 value (ties to the even code), and the next term does the same with what is left over, r - value.  Every step
// is exact in f32, so the bytes can be restated on a CPU.  A block with a NaN or an infinity is NaN as a whole: its first
// scale byte is 255 (E8M0's NaN), its codes are 0, and its later terms are 0.
#include <algorithm>

#include "head.cuh"

namespace dsx {
namespace {

constexpr int kThreads = 256;

// Eight floats -> eight E2M1 codes (round to nearest even, saturating), element i in nibble i.
__device__ __forceinline__ uint32_t e2m1_encode8(const float (&v)[8]) {
    uint32_t out;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(out)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return out;
}

// Eight consecutive values of a row, as f32.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = to_f32(p[j]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float2 f = unpack2<T>(w[j]);
            v[2 * j] = f.x; v[2 * j + 1] = f.y;
        }
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ p, const float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < 8; j++) p[j] = from_f32<T>(v[j]);
    } else if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
}

// max |.| of eight values as f32, NaN if one of them is
__device__ __forceinline__ float abs_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}
__device__ __forceinline__ float abs_max8(const float (&v)[8]) {
    return abs_max_nan(abs_max_nan(abs_max_nan(v[0], v[1]), abs_max_nan(v[2], v[3])), abs_max_nan(abs_max_nan(v[4], v[5]), abs_max_nan(v[6], v[7])));
}

// A lane holds 8 consecutive values, four neighbouring lanes a block of 32: loads are 16 (f32: 32) bytes a lane and coalesced, the
// block's maximum is two shuffles away, and a warp stores 128 bytes of codes.  Groups of 8 are numbered through all rows, so a
// short row wastes no lane; K / 8 is a multiple of 4, so a block never straddles two quads.  ITEMS groups a lane are requested before the
// first is worked on: a full grid (8 blocks of 256 an SM) of one 16-byte load a lane is 32 KB in flight an SM, too little for HBM.
template <int DT, int TERMS, bool VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads)
mxfp4_quantize_kernel(const void* __restrict__ x_, int64_t n_groups, uint32_t groups_per_row, int64_t row_stride, uint32_t* __restrict__ codes,
                      uint8_t* __restrict__ scales) {
    using T = typename Elem<DT>::T;
    pdl_wait();
    if (ITEMS == 1) pdl_launch_dependents();   // a small launch leaves room for the next kernel to set itself up
    const T* __restrict__ x = reinterpret_cast<const T*>(x_);
    const bool dense = row_stride == (int64_t)groups_per_row * 8;
    // n_groups is a multiple of 4, so the four lanes of a block are in range or out of it together; the mask of a quad
    const uint32_t quad = 0xFu << (threadIdx.x & 28u);
    for (int64_t g0 = (int64_t)blockIdx.x * (kThreads * ITEMS) + threadIdx.x; g0 < n_groups; g0 += (int64_t)gridDim.x * (kThreads * ITEMS)) {
        float v[ITEMS][8];
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int64_t g = g0 + i * kThreads;
            int64_t off = g * 8;
            if (!dense) {
                const int64_t row = g / groups_per_row;
                off = row * row_stride + (g - row * groups_per_row) * 8;
            }
            if (g < n_groups) load8<T, VEC>(x + off, v[i]);
        }
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int64_t g = g0 + i * kThreads;
            if (g >= n_groups) break;
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                float m = abs_max8(v[i]);
                m = abs_max_nan(m, __shfl_xor_sync(quad, m, 1));
                m = abs_max_nan(m, __shfl_xor_sync(quad, m, 2));
                const uint32_t amax = __float_as_uint(m);
                const bool bad = amax >= 0x7F800000u;   // infinite or NaN (whose sign bit is clear behind max.NaN)
                const int e = min(max((int)(amax >> 23) - 2 + ((amax & 0x7FFFFFu) > 0x400000u ? 1 : 0), 1), 253);
                const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
                float sv[8];
#pragma unroll
                for (int j = 0; j < 8; j++) sv[j] = v[i][j] * inv;
                const uint32_t w = bad ? 0u : e2m1_encode8(sv);
                codes[(int64_t)t * n_groups + g] = w;
                if ((threadIdx.x & 3u) == 0u) scales[(int64_t)t * (n_groups >> 2) + (g >> 2)] = bad ? 255u : (uint8_t)e;
                if (t + 1 < TERMS) {
                    // value = code * 2^(e - 127): the codes' f32 forms are scaled by 2^-126, hence two exact multiplications
                    const float scl = __uint_as_float((uint32_t)e << 23);
#pragma unroll
                    for (int j = 0; j < 8; j++) v[i][j] = bad ? 0.0f : __fmaf_rn(-e2m1_to_f32(w >> (4 * j)), scl, v[i][j]);   // exact: the residual
                }
            }
        }
    }
}

template <int DT, bool VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads)
mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n_groups, uint32_t groups_per_row, int terms,
                        void* __restrict__ out_, int64_t row_stride) {
    using T = typename Elem<DT>::T;
    pdl_wait();
    if (ITEMS == 1) pdl_launch_dependents();
    T* __restrict__ out = reinterpret_cast<T*>(out_);
    const bool dense = row_stride == (int64_t)groups_per_row * 8;
    for (int64_t g0 = (int64_t)blockIdx.x * (kThreads * ITEMS) + threadIdx.x; g0 < n_groups; g0 += (int64_t)gridDim.x * (kThreads * ITEMS)) {
        float v[ITEMS][8];
        for (int t = 0; t < terms; t++) {
            uint32_t w[ITEMS], e[ITEMS];
#pragma unroll
            for (int i = 0; i < ITEMS; i++) {
                const int64_t g = min(g0 + i * kThreads, n_groups - 1);
                w[i] = __ldg(codes + (int64_t)t * n_groups + g);
                e[i] = __ldg(scales + (int64_t)t * (n_groups >> 2) + (g >> 2));
            }
#pragma unroll
            for (int i = 0; i < ITEMS; i++) {
                const float s = e8m0_value(e[i]);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float d = e2m1_to_f32(w[i] >> (4 * j)) * s;
                    v[i][j] = t == 0 ? d : v[i][j] + d;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int64_t g = g0 + i * kThreads;
            if (g >= n_groups) break;
            int64_t off = g * 8;
            if (!dense) {
                const int64_t row = g / groups_per_row;
                off = row * row_stride + (g - row * groups_per_row) * 8;
            }
            store8<T, VEC>(out + off, v[i]);
        }
    }
}

// Launches `small` (a group a lane, at most 8 blocks an SM) or, where that would go round more than once, `large` (four groups).
template <typename K, typename... A>
int launch_rows(K small, K large, int64_t n_groups, cudaStream_t s, A... args) {
    int sms = 0;
    if (int rc = head_sm_count(&sms)) return rc;
    const int64_t cap = (int64_t)sms * 8, blocks = (n_groups + kThreads - 1) / kThreads;
    const bool big = blocks > cap;
    DSX_CUDA(launch_pdl(big ? large : small, dim3((unsigned)(big ? std::min(cap, (blocks + 3) / 4) : blocks)), dim3(kThreads), 0, s, args...));
    DSX_LAUNCHED();
    return DSX_OK;
}

template <int DT, bool VEC, int TERMS>
int launch_quantize(cudaStream_t s, const void* x, int64_t n_groups, uint32_t gpr, int64_t stride, uint32_t* codes, uint8_t* scales) {
    return launch_rows(mxfp4_quantize_kernel<DT, TERMS, VEC, 1>, mxfp4_quantize_kernel<DT, TERMS, VEC, 4>, n_groups, s, x, n_groups, gpr, stride, codes, scales);
}
template <int DT, bool VEC>
int launch_quantize_terms(int terms, cudaStream_t s, const void* x, int64_t n_groups, uint32_t gpr, int64_t stride, uint32_t* codes, uint8_t* scales) {
    if (terms == 1) return launch_quantize<DT, VEC, 1>(s, x, n_groups, gpr, stride, codes, scales);
    if (terms == 2) return launch_quantize<DT, VEC, 2>(s, x, n_groups, gpr, stride, codes, scales);
    return launch_quantize<DT, VEC, 3>(s, x, n_groups, gpr, stride, codes, scales);
}

int check_rows(const char* what, int dtype, int64_t rows, int64_t k, int64_t row_stride, int n_terms) {
    DSX_REQUIRE(dtype_ok(dtype), "%s: unknown element type %d", what, dtype);
    DSX_REQUIRE(rows >= 0 && k >= 32 && k % 32 == 0 && k <= ((int64_t)1 << 30), "%s: %lld rows of %lld columns (a multiple of 32)", what, (long long)rows,
                (long long)k);
    DSX_REQUIRE(n_terms >= 1 && n_terms <= 3, "%s: %d terms (1 to 3)", what, n_terms);
    DSX_REQUIRE(row_stride >= k || rows <= 1, "%s: row stride %lld below the %lld columns of a row", what, (long long)row_stride, (long long)k);
    return DSX_OK;
}

}  // namespace
}  // namespace dsx

using namespace dsx;

extern "C" {

int dsx_mxfp4_quantize(const void* x, int dtype, int64_t rows, int64_t k, int64_t row_stride, int n_terms, void* codes, void* scales, dsx_stream_t stream) {
    if (int rc = check_rows("mxfp4_quantize", dtype, rows, k, row_stride, n_terms)) return rc;
    if (rows == 0) return DSX_OK;
    DSX_REQUIRE(x && codes && scales, "mxfp4_quantize: null argument");
    DSX_REQUIRE(((uintptr_t)x & (dtype_size(dtype) - 1)) == 0 && ((uintptr_t)codes & 15) == 0, "mxfp4_quantize: x must be aligned to its elements, codes to 16 bytes");
    const int64_t n_groups = rows * (k / 8);
    const bool vec = (((uintptr_t)x | (uintptr_t)(rows > 1 ? row_stride * dtype_size(dtype) : 0)) & 15) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT)                                                                                                                                \
    return vec ? launch_quantize_terms<DT, true>(n_terms, s, x, n_groups, (uint32_t)(k / 8), row_stride, (uint32_t*)codes, (uint8_t*)scales)        \
               : launch_quantize_terms<DT, false>(n_terms, s, x, n_groups, (uint32_t)(k / 8), row_stride, (uint32_t*)codes, (uint8_t*)scales)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    DSX_GO(DSX_F16);
#undef DSX_GO
}

int dsx_mxfp4_dequantize(const void* codes, const void* scales, int64_t rows, int64_t k, int n_terms, void* out, int dtype, int64_t row_stride,
                         dsx_stream_t stream) {
    if (int rc = check_rows("mxfp4_dequantize", dtype, rows, k, row_stride, n_terms)) return rc;
    if (rows == 0) return DSX_OK;
    DSX_REQUIRE(codes && scales && out, "mxfp4_dequantize: null argument");
    DSX_REQUIRE(((uintptr_t)out & (dtype_size(dtype) - 1)) == 0 && ((uintptr_t)codes & 15) == 0,
                "mxfp4_dequantize: out must be aligned to its elements, codes to 16 bytes");
    const int64_t n_groups = rows * (k / 8);
    const bool vec = (((uintptr_t)out | (uintptr_t)(rows > 1 ? row_stride * dtype_size(dtype) : 0)) & 15) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
    const uint32_t* c = (const uint32_t*)codes;
    const uint8_t* e = (const uint8_t*)scales;
    const uint32_t gpr = (uint32_t)(k / 8);
#define DSX_GO(DT)                                                                                                                                \
    return vec ? launch_rows(mxfp4_dequantize_kernel<DT, true, 1>, mxfp4_dequantize_kernel<DT, true, 4>, n_groups, s, c, e, n_groups, gpr, n_terms, out, row_stride) \
               : launch_rows(mxfp4_dequantize_kernel<DT, false, 1>, mxfp4_dequantize_kernel<DT, false, 4>, n_groups, s, c, e, n_groups, gpr, n_terms, out, row_stride)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    DSX_GO(DSX_F16);
#undef DSX_GO
}

}  // extern "C"
