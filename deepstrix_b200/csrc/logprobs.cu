// Log probabilities of given tokens, entropy and the most likely alternatives, from rows of logits.
#include "head.cuh"

namespace dsx {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_max(float v, float* s) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s[0];
    for (int i = 1; i < kThreads / 32; i++) v = fmaxf(v, s[i]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ float block_sum(float v, float* s) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < kThreads / 32; i++) v += s[i];
    __syncthreads();
    return v;
}

// A block per row: one pass for the maximum, one for the sums, one per alternative.
template <int DT>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const void* __restrict__ logits, int64_t V, int64_t row_stride, float scale, const int32_t* __restrict__ tokens, int n_given,
                      float* __restrict__ logprobs, float* __restrict__ entropy, int n_alt, int32_t* __restrict__ alts, float* __restrict__ alt_logprobs) {
    using T = typename Elem<DT>::T;
    __shared__ float s_red[kThreads / 32];
    __shared__ unsigned long long s_best;
    const int64_t t = blockIdx.x;
    const T* row = reinterpret_cast<const T*>(logits) + t * row_stride;
    float m = -INFINITY, bad = 0.0f;
    for (int64_t i = threadIdx.x; i < V; i += kThreads) {
        const float x = to_f32(row[i]);
        if (!(x <= 3.402823466e38f)) bad = 1.0f;   // NaN or +inf
        m = fmaxf(m, x);
    }
    m = block_max(m, s_red);
    bad = block_max(bad, s_red);
    const bool empty = m == -INFINITY;
    const float mm = empty ? 0.0f : m;
    float s = 0.0f, u = 0.0f;
    if (bad == 0.0f)
        for (int64_t i = threadIdx.x; i < V; i += kThreads) {
            const float d = (to_f32(row[i]) - mm) * scale, e = expf(d);
            s += e;
            if (e > 0.0f) u += d * e;
        }
    s = block_sum(s, s_red);
    u = block_sum(u, s_red);
    const float log_s = empty ? 0.0f : logf(s), nan = __uint_as_float(0x7FC00000u);
    auto logp = [&](float x) { return bad != 0.0f ? nan : (x - mm) * scale - log_s; };
    for (int g = threadIdx.x; g < n_given; g += kThreads) {
        const int32_t tok = tokens[t * n_given + g];
        logprobs[t * n_given + g] = tok >= 0 && tok < V ? logp(to_f32(row[tok])) : -INFINITY;
    }
    if (threadIdx.x == 0 && entropy != nullptr) entropy[t] = bad != 0.0f ? nan : (empty ? 0.0f : log_s - u / s);
    unsigned long long last = ~0ull;
    for (int a = 0; a < n_alt; a++) {
        if (threadIdx.x == 0) s_best = 0ull;
        __syncthreads();
        unsigned long long best = 0ull;   // (ordered value, inverted index) of the largest entry below `last`
        if (bad == 0.0f)
            for (int64_t i = threadIdx.x; i < V; i += kThreads) {
                const float x = to_f32(row[i]) + 0.0f;
                if (x == -INFINITY) continue;
                const uint32_t b = __float_as_uint(x), o = (b & 0x80000000u) ? ~b : b | 0x80000000u;
                const unsigned long long key = ((unsigned long long)o << 32) | (uint32_t)~(uint32_t)i;
                if (key < last && key > best) best = key;
            }
        atomicMax(&s_best, best);
        __syncthreads();
        last = s_best;
        __syncthreads();
        if (threadIdx.x == 0) {
            const int32_t id = last ? (int32_t)~(uint32_t)last : -1;
            alts[t * n_alt + a] = id;
            alt_logprobs[t * n_alt + a] = id >= 0 ? logp(to_f32(row[id])) : (bad != 0.0f ? nan : -INFINITY);
        }
        if (last == 0ull) last = 1ull;
    }
}

}  // namespace
}  // namespace dsx

using namespace dsx;

extern "C" int dsx_token_logprobs(const void* logits, int dtype, int64_t t, int64_t v, int64_t row_stride, float inv_temperature, const int32_t* tokens,
                                  int n_given, float* logprobs, float* entropy, int n_alt, int32_t* alts, float* alt_logprobs, dsx_stream_t stream) {
    DSX_REQUIRE(dtype_ok(dtype), "token_logprobs: unknown element type %d", dtype);
    DSX_REQUIRE(t >= 0 && t <= 0x7FFFFFFF && v >= 1 && v <= 0x7FFFFFFF, "token_logprobs: %lld rows of %lld logits", (long long)t, (long long)v);
    DSX_REQUIRE(n_given >= 0 && n_given <= 1024 && n_alt >= 0 && n_alt <= 32, "token_logprobs: %d given tokens (at most 1024), %d alternatives (at most 32)",
                n_given, n_alt);
    DSX_REQUIRE(inv_temperature > 0.0f && inv_temperature <= 1.0e6f, "token_logprobs: inverse temperature %g (above 0, at most 1e6)", inv_temperature);
    if (t == 0) return DSX_OK;
    DSX_REQUIRE(row_stride >= v || t == 1, "token_logprobs: row stride %lld below the %lld logits of a row", (long long)row_stride, (long long)v);
    DSX_REQUIRE(logits && (n_given == 0 || (tokens && logprobs)) && (n_alt == 0 || (alts && alt_logprobs)), "token_logprobs: null argument");
    DSX_REQUIRE(((uintptr_t)logits & (dtype_size(dtype) - 1)) == 0, "token_logprobs: logits must be aligned to their elements");
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT)                                                                                                                                  \
    token_logprobs_kernel<DT><<<(unsigned)t, kThreads, 0, s>>>(logits, v, row_stride, inv_temperature, tokens, n_given, logprobs, entropy, n_alt, alts, \
                                                               alt_logprobs)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    else if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    else DSX_GO(DSX_F16);
#undef DSX_GO
    DSX_LAUNCHED();
    return DSX_OK;
}
