// out[m, n] = sum over terms and k of A_term[m, k] * W[n, k], both operands MXFP4 rows, f32 accumulation, one rounding.
#include "head.cuh"

namespace dsx {
namespace {

constexpr int kTile = 64;

// 64 x 64 outputs a block, 4 x 4 a thread; 32 columns (one scale block) of both operands expanded to f32 in shared memory a step.
template <int DT>
__global__ void __launch_bounds__(256)
mxfp4_matmul_kernel(const uint32_t* __restrict__ a_codes, const uint8_t* __restrict__ a_scales, int terms, int64_t M, const uint32_t* __restrict__ w_codes,
                    const uint8_t* __restrict__ w_scales, int64_t N, int64_t K, void* __restrict__ out_, int64_t row_stride) {
    using T = typename Elem<DT>::T;
    __shared__ float sa[32][kTile + 1], sw[32][kTile + 1];
    const int64_t n0 = (int64_t)blockIdx.x * kTile, m0 = (int64_t)blockIdx.y * kTile;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t words = K / 8, blocks = K / 32;
    float acc[4][4] = {};
    for (int64_t b = 0; b < blocks; b++) {
        {   // thread = (row tid / 4, eight columns (tid % 4))
            const int r = tid >> 2, c = tid & 3;
            float v[8] = {};
            if (m0 + r < M)
                for (int t = 0; t < terms; t++) {
                    const int64_t row = (int64_t)t * M + m0 + r;
                    const uint32_t w = a_codes[row * words + b * 4 + c];
                    const float s = e8m0_value(a_scales[row * blocks + b]);
                    for (int j = 0; j < 8; j++) v[j] += e2m1_to_f32(w >> (4 * j)) * s;
                }
            for (int j = 0; j < 8; j++) sa[c * 8 + j][r] = v[j];
            float u[8] = {};
            if (n0 + r < N) {
                const uint32_t w = w_codes[(n0 + r) * words + b * 4 + c];
                const float s = e8m0_value(w_scales[(n0 + r) * blocks + b]);
                for (int j = 0; j < 8; j++) u[j] = e2m1_to_f32(w >> (4 * j)) * s;
            }
            for (int j = 0; j < 8; j++) sw[c * 8 + j][r] = u[j];
        }
        __syncthreads();
        for (int k = 0; k < 32; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) acc[i][j] = __fmaf_rn(sa[k][ty * 4 + i], sw[k][tx + 16 * j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            const int64_t m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
            if (m < M && n < N) reinterpret_cast<T*>(out_)[m * row_stride + n] = from_f32<T>(acc[i][j]);
        }
}

}  // namespace
}  // namespace dsx

using namespace dsx;

extern "C" int dsx_mxfp4_matmul(const void* a_codes, const void* a_scales, int n_terms, int64_t m, const void* w_codes, const void* w_scales, int64_t n,
                                int64_t k, void* out, int dtype, int64_t row_stride, dsx_stream_t stream) {
    DSX_REQUIRE(dtype_ok(dtype), "mxfp4_matmul: unknown element type %d", dtype);
    DSX_REQUIRE(m >= 0 && n >= 0 && k >= 32 && k % 32 == 0 && m < ((int64_t)1 << 22) && n < ((int64_t)1 << 31) && k <= ((int64_t)1 << 30),
                "mxfp4_matmul: %lld x %lld x %lld (k a multiple of 32)", (long long)m, (long long)n, (long long)k);
    DSX_REQUIRE(n_terms >= 1 && n_terms <= 3, "mxfp4_matmul: %d terms (1 to 3)", n_terms);
    if (m == 0 || n == 0) return DSX_OK;
    DSX_REQUIRE(a_codes && a_scales && w_codes && w_scales && out, "mxfp4_matmul: null argument");
    DSX_REQUIRE(row_stride >= n || m == 1, "mxfp4_matmul: row stride %lld below the %lld columns of a row", (long long)row_stride, (long long)n);
    DSX_REQUIRE((((uintptr_t)a_codes | (uintptr_t)w_codes) & 15) == 0 && ((uintptr_t)out & (dtype_size(dtype) - 1)) == 0,
                "mxfp4_matmul: codes must be 16-byte aligned, out aligned to its elements");
    const dim3 grid((unsigned)((n + kTile - 1) / kTile), (unsigned)((m + kTile - 1) / kTile));
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT)                                                                                                                              \
    mxfp4_matmul_kernel<DT><<<grid, 256, 0, s>>>((const uint32_t*)a_codes, (const uint8_t*)a_scales, n_terms, m, (const uint32_t*)w_codes,       \
                                                 (const uint8_t*)w_scales, n, k, out, row_stride)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    else if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    else DSX_GO(DSX_F16);
#undef DSX_GO
    DSX_LAUNCHED();
    return DSX_OK;
}
