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
//
// Both directions are bound by HBM where there is one term (65536 x 2048 f32: 89 us to codes, 6.8 TB/s, 98 us back, 6.2; bf16 53 and 55 us), and
// by latency below a megabyte (2 us).  More terms: 8192 x 4096 bf16 15 and 15 us with one, 33 and 28 with three, where the bytes want 18.4.
// Counters of 32768 x 4096 bf16 with three (124 and 104 us, bytes 74): the quantiser issues in 71 % of the clocks (integer pipe 69 %, the
// largest stalls waits for that pipe and for loads) with 37 warps an SM, 40 registers a thread allowing 12 blocks of the 16 its grid
// has an SM, so that the last quarter of them runs by itself; the dequantiser issues in 82 % (integer pipe 77 %) with 26 warps (72 registers).
#include <algorithm>

#include "head.cuh"

namespace dsx {
namespace {

constexpr int kThreads = 128;

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

// N consecutive values of a row, as f32, in 16-byte loads where they are aligned.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void load_values(const T* __restrict__ p, float (&v)[N]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int j = 0; j < N; j++) v[j] = to_f32(p[j]);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p) + i);
            v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 8; i++) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + i);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = unpack2<T>(w[j]);
                v[8 * i + 2 * j] = f.x; v[8 * i + 2 * j + 1] = f.y;
            }
        }
    }
}

// |.| compared with a NaN winning
__device__ __forceinline__ float abs_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
    return r;
}

// A lane holds PER consecutive values -- 8 f32 or 16 of 16 bits, 32 bytes -- so four or two neighbouring lanes make a block of 32: loads
// are coalesced, the block's maximum is a shuffle or two away, and what a block costs beside its values is shared by as many as registers
// allow.  Units of PER are numbered through all rows, so a short row wastes no lane; a block never straddles two quads or pairs.  48 KB
// of loads are in flight an SM.
template <int DT> constexpr int kPer = DT == DSX_F32 ? 8 : 16;

template <int DT, int TERMS, bool VEC>
__global__ void __launch_bounds__(kThreads)
mxfp4_quantize_kernel(const void* __restrict__ x_, int64_t n_units, uint32_t units_per_row, int64_t row_stride, uint32_t* __restrict__ codes,
                      uint8_t* __restrict__ scales, int release) {
    using T = typename Elem<DT>::T;
    constexpr int PER = kPer<DT>, LANES = 32 / PER;   // of a block
    pdl_wait();
    // A small launch leaves room for the next kernel to set itself up.  What comes after the wait is all this kernel writes, and no kernel of
    // the library reads codes before its own wait.
    if (release) pdl_launch_dependents();
    const T* __restrict__ x = reinterpret_cast<const T*>(x_);
    const bool dense = row_stride == (int64_t)units_per_row * PER;
    // n_units is a multiple of LANES, so the lanes of a block are in range or out of it together; their mask
    const uint32_t mates = ((1u << LANES) - 1u) << (threadIdx.x & (32u - LANES));
    for (int64_t g = (int64_t)blockIdx.x * kThreads + threadIdx.x; g < n_units; g += (int64_t)gridDim.x * kThreads) {
        int64_t off = g * PER;
        if (!dense) {
            const int64_t row = g / units_per_row;
            off = row * row_stride + (g - row * units_per_row) * PER;
        }
        float v[PER];
        load_values<T, VEC, PER>(x + off, v);
        bool bad = false;
#pragma unroll
        for (int t = 0; t < TERMS; t++) {
            float m = abs_max_nan(v[0], v[1]);
#pragma unroll
            for (int j = 2; j < PER; j++) m = abs_max_nan(m, v[j]);
#pragma unroll
            for (int o = 1; o < LANES; o *= 2) m = abs_max_nan(m, __shfl_xor_sync(mates, m, o));
            const uint32_t amax = __float_as_uint(m);
            if (t == 0) bad = amax >= 0x7F800000u;   // infinite or NaN (whose sign bit is clear behind max.NaN)
            const int e = min(max((int)(amax >> 23) - 2 + ((amax & 0x7FFFFFu) > 0x400000u ? 1 : 0), 1), 253);
            const float inv = __uint_as_float((uint32_t)(254 - e) << 23), scl = __uint_as_float((uint32_t)e << 23);
            const uint64_t inv2 = pair(inv, inv), minus_scl2 = pair(-scl, -scl);
            uint32_t w[PER / 8];
#pragma unroll
            for (int i = 0; i < PER / 8; i++) {
                float sv[8];
#pragma unroll
                for (int j = 0; j < 8; j += 2) unpair(mul2(pair(v[8 * i + j], v[8 * i + j + 1]), inv2), sv[j], sv[j + 1]);
                const uint32_t c = e2m1_encode8(sv);
                w[i] = bad ? 0u : c;
                if (t + 1 < TERMS) {
                    // Adding +0 makes minus zero plain zero, as in the CPU quantiser's integer table: the sign of a zero residual, and with it the
                    // next term's code, is the same there.  (In a bad block the rest is as bad, and its codes are 0 from here on.)
                    float d[8];
                    e2m1_values(c, d);
#pragma unroll
                    for (int j = 0; j < 8; j += 2)   // exact: the residual
                        unpair(fma2(add2(pair(d[j], d[j + 1]), pair(0.0f, 0.0f)), minus_scl2, pair(v[8 * i + j], v[8 * i + j + 1])), v[8 * i + j], v[8 * i + j + 1]);
                }
            }
            uint32_t* to = codes + ((int64_t)t * n_units + g) * (PER / 8);
            if constexpr (PER == 16) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
            else *to = w[0];
            if ((threadIdx.x & (LANES - 1)) == 0) scales[((int64_t)t * n_units + g) / LANES] = bad ? (t == 0 ? 255u : 1u) : (uint8_t)e;
        }
    }
}

// A lane makes 16 bytes of the result (4 f32 or 8 values of 16 bits), so that a warp's stores are whole sectors; ITEMS of them, whose codes
// and scales -- a few bytes a lane -- are requested together.
template <int DT> constexpr int kOut = DT == DSX_F32 ? 4 : 8;

template <int DT, int TERMS, bool VEC, int ITEMS>
__global__ void __launch_bounds__(kThreads)
mxfp4_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int64_t n_units, uint32_t units_per_row,
                        void* __restrict__ out_, int64_t row_stride) {
    using T = typename Elem<DT>::T;
    constexpr int PER = kOut<DT>, LANES = 32 / PER;
    pdl_wait();   // and no early release: the result may be router weights, which the router copies before its own wait
    T* __restrict__ out = reinterpret_cast<T*>(out_);
    const bool dense = row_stride == (int64_t)units_per_row * PER;
    for (int64_t g0 = (int64_t)blockIdx.x * (kThreads * ITEMS) + threadIdx.x; g0 < n_units; g0 += (int64_t)gridDim.x * (kThreads * ITEMS)) {
        uint32_t w[ITEMS][TERMS], e[ITEMS][TERMS];
#pragma unroll
        for (int i = 0; i < ITEMS; i++)
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                const int64_t g = (int64_t)t * n_units + min(g0 + i * kThreads, n_units - 1);
                w[i][t] = PER == 8 ? __ldg(reinterpret_cast<const uint32_t*>(codes) + g) : (uint32_t)__ldg(reinterpret_cast<const uint16_t*>(codes) + g);
                e[i][t] = __ldg(scales + g / LANES);
            }
#pragma unroll
        for (int i = 0; i < ITEMS; i++) {
            const int64_t g = g0 + i * kThreads;
            if (g >= n_units) break;
            float v[PER];
#pragma unroll
            for (int t = 0; t < TERMS; t++) {
                const float s = e8m0_value(e[i][t]);
                float d[PER];
                e2m1_values(w[i][t], d);
#pragma unroll
                for (int j = 0; j < PER; j += 2) {   // the product is exact
                    const uint64_t p = pair(d[j], d[j + 1]), s2 = pair(s, s);
                    unpair(t == 0 ? mul2(p, s2) : fma2(p, s2, pair(v[j], v[j + 1])), v[j], v[j + 1]);
                }
            }
            int64_t off = g * PER;
            if (!dense) {
                const int64_t row = g / units_per_row;
                off = row * row_stride + (g - row * units_per_row) * PER;
            }
            if constexpr (!VEC) {
#pragma unroll
                for (int j = 0; j < PER; j++) out[off + j] = from_f32<T>(v[j]);
            } else if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4*>(out + off) = make_float4(v[0], v[1], v[2], v[3]);
            } else {
                *reinterpret_cast<uint4*>(out + off) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
            }
        }
    }
}

constexpr int kPerSm = 2048 / kThreads;   // blocks of a grid an SM; what is resident at once is less where a thread has more than 32 registers (down to 7)

template <typename K, typename... A>
int launch_rows(K kernel, int64_t blocks, cudaStream_t s, A... args) {
    DSX_CUDA(launch_pdl(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, s, args...));
    DSX_LAUNCHED();
    return DSX_OK;
}

template <int DT, bool VEC>
int launch_quantize(int terms, cudaStream_t s, const void* x, int64_t rows, int64_t k, int64_t stride, uint32_t* codes, uint8_t* scales) {
    const int64_t n = rows * (k / kPer<DT>);
    const uint32_t per_row = (uint32_t)(k / kPer<DT>);
    int sms = 0;
    if (int rc = head_sm_count(&sms)) return rc;
    const int64_t cap = (int64_t)sms * kPerSm, blocks = std::min(cap, (n + kThreads - 1) / kThreads);
    const int release = blocks <= cap / 4;
    if (terms == 1) return launch_rows(mxfp4_quantize_kernel<DT, 1, VEC>, blocks, s, x, n, per_row, stride, codes, scales, release);
    if (terms == 2) return launch_rows(mxfp4_quantize_kernel<DT, 2, VEC>, blocks, s, x, n, per_row, stride, codes, scales, release);
    return launch_rows(mxfp4_quantize_kernel<DT, 3, VEC>, blocks, s, x, n, per_row, stride, codes, scales, release);
}

template <int DT, int TERMS, bool VEC>
int launch_dequantize_terms(cudaStream_t s, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, void* out, int64_t stride) {
    const int64_t n = rows * (k / kOut<DT>);
    const uint32_t per_row = (uint32_t)(k / kOut<DT>);
    int sms = 0;
    if (int rc = head_sm_count(&sms)) return rc;
    // four items a lane once there are more than one for every lane of sixteen blocks an SM, and more blocks than that (65536 x 2048 to bf16 in an
    // earlier build: 65 us, 70 us in a grid of sixteen an SM; two items 68, one 81)
    const int64_t lanes = (int64_t)sms * kPerSm * kThreads;
    if (n <= lanes) return launch_rows(mxfp4_dequantize_kernel<DT, TERMS, VEC, 1>, (n + kThreads - 1) / kThreads, s, codes, scales, n, per_row, out, stride);
    const int64_t blocks = std::min<int64_t>((n + 4 * kThreads - 1) / (4 * kThreads), 4 * sms * kPerSm);
    return launch_rows(mxfp4_dequantize_kernel<DT, TERMS, VEC, 4>, blocks, s, codes, scales, n, per_row, out, stride);
}
template <int DT, bool VEC>
int launch_dequantize(int terms, cudaStream_t s, const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t k, void* out, int64_t stride) {
    if (terms == 1) return launch_dequantize_terms<DT, 1, VEC>(s, codes, scales, rows, k, out, stride);
    if (terms == 2) return launch_dequantize_terms<DT, 2, VEC>(s, codes, scales, rows, k, out, stride);
    return launch_dequantize_terms<DT, 3, VEC>(s, codes, scales, rows, k, out, stride);
}

int check_rows(const char* what, int dtype, int64_t rows, int64_t k, int64_t row_stride, int n_terms) {
    DSX_REQUIRE(dtype_ok(dtype), "%s: unknown element type %d", what, dtype);
    DSX_REQUIRE(k >= 32 && k % 32 == 0 && k <= ((int64_t)1 << 30) && rows >= 0 && rows <= ((int64_t)1 << 46) / k,
                "%s: %lld rows of %lld columns (a multiple of 32, at most 2^30; 2^46 values)", what, (long long)rows, (long long)k);
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
    const bool vec = (((uintptr_t)x | (uintptr_t)(rows > 1 ? row_stride * dtype_size(dtype) : 0)) & 15) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT)                                                                                                        \
    return vec ? launch_quantize<DT, true>(n_terms, s, x, rows, k, row_stride, (uint32_t*)codes, (uint8_t*)scales)          \
               : launch_quantize<DT, false>(n_terms, s, x, rows, k, row_stride, (uint32_t*)codes, (uint8_t*)scales)
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
    const bool vec = (((uintptr_t)out | (uintptr_t)(rows > 1 ? row_stride * dtype_size(dtype) : 0)) & 15) == 0;
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT)                                                                                                                \
    return vec ? launch_dequantize<DT, true>(n_terms, s, (const uint8_t*)codes, (const uint8_t*)scales, rows, k, out, row_stride)   \
               : launch_dequantize<DT, false>(n_terms, s, (const uint8_t*)codes, (const uint8_t*)scales, rows, k, out, row_stride)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    DSX_GO(DSX_F16);
#undef DSX_GO
}

}  // extern "C"
