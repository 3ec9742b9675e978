// Log probabilities of given tokens, entropy and the most likely alternatives, from rows of logits, in one pass over them.
//
// With z = logit * scale, m the row's largest logit, d = (logit - m) * scale:   s = sum e^d,   u = sum d e^d,
//   log p(token) = d(token) - ln s,   entropy = ln s - u / s,   alternatives = the n_alt largest logits (equal logits: lower index).
// Counterparts in the reference (paths relative to the deepstrix repository): its sampler's softmax over the vocabulary
// (crates/v4flash-kernels/kernels/softmax_sample.hip) and the teacher-forced scoring of tests/v41_golden_gate.rs.
//
// One pass.  A thread keeps its own running maximum and its s and u relative to it; it takes 32 bytes of logits at a time and rescales
// only when their maximum is new, so an element costs about one conversion, one subtraction, one exponential and three
// multiply-adds.  The alternatives ride on the same maximum: a chunk is looked at again only when its largest logit reaches the
// block's threshold, a value that at least n_alt logits of the row are known to reach.  What reaches it goes to the warp's candidate list
// in shared memory; 32 candidates at a time are sorted in registers and merged into the warp's best 32 (one key per lane), whose
// n_alt-th becomes the new threshold.  A sorted row that beats the threshold at every element is slow, but right.
// A row belongs to one block, or, when there are few rows, to the blocks of a cluster that join their sums and lists through
// distributed shared memory: one launch, no workspace, and the order of every addition is fixed.
//
// Bound: HBM for f32 and for short lists; bf16 and f16 rows at full HBM rate are 11.6 elements a clock and SM, of which the exponentials
// take 16 lanes a clock -- so the instruction count above is what matters there.
#include <algorithm>

#include "head.cuh"

namespace dsx {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxAlt = 32;            // one per lane of the warp that holds a list
constexpr int kMaxCluster = 8;
constexpr float kLowest = -3.402823466e38f;
constexpr uint32_t kFloor = 0x00800000u;   // order_of(kLowest): nothing finite is below it
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// 2^x; the instruction is off by at most 2 ulp, and 0 for x below -150
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// the larger of two, NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Logits compare as (value descending, index ascending): value bits mapped to an ascending unsigned order above the inverted index.  The
// smallest key, 0, is "nothing"; a masked logit (-inf) is never made into a key.
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // -0 ties with 0
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) { return ((uint64_t)order_of(x) << 32) | (uint32_t)~i; }

// Descending bitonic sort of one key a lane.
__device__ __forceinline__ uint64_t sort32(uint64_t k, int lane) {
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int j = size >> 1; j > 0; j >>= 1) {
            const uint64_t o = __shfl_xor_sync(0xFFFFFFFFu, k, j);
            const bool up = ((lane & size) != 0) != ((lane & j) != 0);   // this lane keeps the smaller one
            k = up ? (k < o ? k : o) : (k > o ? k : o);
        }
    return k;
}
// The best 32 of two descending lists, descending.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b, int lane) {
    const uint64_t r = __shfl_sync(0xFFFFFFFFu, b, 31 - lane);
    uint64_t k = a > r ? a : r;   // bitonic: the larger half
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) {
        const uint64_t o = __shfl_xor_sync(0xFFFFFFFFu, k, j);
        k = (lane & j) ? (k < o ? k : o) : (k > o ? k : o);
    }
    return k;
}

// s and u relative to m: sums of 2^t and t 2^t with t = (x - m) * c.
struct Sums {
    float m, s, u;
    // to a larger maximum; s = 0 (nothing yet) stays 0 whatever the difference
    __device__ __forceinline__ void raise(float to, float c) {
        const float t = fmaxf((m - to) * c, -200.0f), e = exp2_fast(t);
        u = (u + s * t) * e;
        s *= e;
        m = to;
    }
    __device__ __forceinline__ void add(Sums o, float c) {
        const float to = fmaxf(m, o.m);
        raise(to, c);
        o.raise(to, c);
        s += o.s;
        u += o.u;
    }
};

template <typename T> struct Chunk;   // 32 bytes: 8 floats or 16 halves
template <> struct Chunk<float> { static constexpr int n = 8; };
template <> struct Chunk<__nv_bfloat16> { static constexpr int n = 16; };
template <> struct Chunk<__half> { static constexpr int n = 16; };

struct Shared {
    uint32_t threshold;                     // order of a value that n_alt logits of the row reach (kFloor: any)
    int pending[kWarps];                    // candidates on the warps' lists
    Sums sums[kWarps];
    uint64_t best[kWarps][32];
    Sums block_sums;
    float stats[2];                         // the row's m and ln s
};

template <int DT>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const void* __restrict__ logits, int64_t T_rows, int64_t V, int64_t row_stride, float scale, const int32_t* __restrict__ tokens,
                      int n_given, float* __restrict__ logprobs, float* __restrict__ entropy, int n_alt, int32_t* __restrict__ alts,
                      float* __restrict__ alt_logprobs, int splits) {
    using T = typename Elem<DT>::T;
    constexpr int kChunk = Chunk<T>::n;
    constexpr int kList = 64 + 32 * kChunk;     // candidates of a warp: fewer than 32 left over, a chunk of every lane, the elements at the edges
    extern __shared__ uint64_t s_list[];        // [warps][kList]
    __shared__ Shared sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = splits > 1 ? blockIdx.x % splits : 0;
    const float c = scale * kLog2e;
    uint64_t* list = s_list + (size_t)warp * kList;

    for (int64_t row = blockIdx.x / splits; row < T_rows; row += gridDim.x / splits) {
        const T* __restrict__ x = reinterpret_cast<const T*>(logits) + row * row_stride;
        if (threadIdx.x == 0) sh.threshold = kFloor;
        if (threadIdx.x < kWarps) sh.pending[threadIdx.x] = 0;
        __syncthreads();
        // whole 16-byte words from the row's first aligned element on; the few elements before and after them one by one
        const int head = (int)min((int64_t)(((16u - (uint32_t)((uintptr_t)x & 15u)) & 15u) / sizeof(T)), V);
        const int64_t n_chunks = (V - head) / kChunk;
        const int64_t body = head + n_chunks * kChunk;
        Sums a{kLowest, 0.0f, 0.0f};
        uint64_t mine = 0ull;                   // the warp's best, descending over its lanes
        uint32_t own = kFloor;                  // lowest order that may still enter that list, for elements behind those in it
        auto flush = [&](bool all) {            // merge candidates 32 at a time; the rest stays (or goes too, padded with nothing)
            int pending = *(volatile int*)&sh.pending[warp];
            if (!all && pending < 32) return;
            while (pending >= 32 || (all && pending > 0)) {
                const int n = min(pending, 32);
                const uint64_t k = lane < n ? list[pending - n + lane] : 0ull;
                pending -= n;
                mine = merge32(mine, sort32(k, lane), lane);
            }
            __syncwarp();
            const uint32_t kth = (uint32_t)(__shfl_sync(0xFFFFFFFFu, mine, n_alt - 1) >> 32);
            if (lane == 0) {
                sh.pending[warp] = pending;
                if (kth != 0u) atomicMax(&sh.threshold, kth);
            }
            if (kth != 0u) own = kth + 1u;      // what comes later has a higher index: an equal logit loses
            __syncwarp();
        };
        auto load = [&](int64_t ch, uint32_t (&w)[8]) {
            const uint4* p = reinterpret_cast<const uint4*>(x + head + ch * kChunk);
            const uint4 w0 = __ldg(p), w1 = __ldg(p + 1);
            w[0] = w0.x; w[1] = w0.y; w[2] = w0.z; w[3] = w0.w; w[4] = w1.x; w[5] = w1.y; w[6] = w1.z; w[7] = w1.w;
        };
        // every warp takes whole rounds, so that its votes are complete; the next round's logits are requested before this one's work
        const int64_t per_round = (int64_t)kThreads * splits;
        const int64_t ch0 = (int64_t)rank * kThreads + threadIdx.x;
        uint32_t next[8];
        if (ch0 < n_chunks) load(ch0, next);
        for (int64_t ch = ch0; ch - lane < n_chunks; ch += per_round) {
            const bool live = ch < n_chunks;
            float v[kChunk];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = __uint_as_float(next[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float2 f = unpack2<T>(next[j]);
                    v[2 * j] = f.x;
                    v[2 * j + 1] = f.y;
                }
            }
            if (ch + per_round < n_chunks) load(ch + per_round, next);
            float top = v[0];
#pragma unroll
            for (int j = 1; j < kChunk; j++) top = fmaxf(top, v[j]);
            if (live) {
                if (top > a.m) a.raise(top, c);
#pragma unroll
                for (int j = 0; j < kChunk; j++) {
                    const float t = max_nan((v[j] - a.m) * c, -200.0f), e = exp2_fast(t);
                    a.s += e;
                    a.u = fmaf(t, e, a.u);
                }
            }
            if (n_alt > 0) {
                uint32_t bound = max(own, *(volatile uint32_t*)&sh.threshold);
                if (ch == ch0) {   // first round: n_alt of the 32 chunks reach the n_alt-th largest of their maxima
                    const uint64_t k = sort32(live && top >= kLowest ? (uint64_t)order_of(top) : 0ull, lane);
                    bound = max(bound, (uint32_t)__shfl_sync(0xFFFFFFFFu, k, n_alt - 1));
                    if (lane == 0) atomicMax(&sh.threshold, bound);
                }
                const float least = value_of(bound);
                if (__any_sync(0xFFFFFFFFu, live && top >= least)) {
                    if (live && top >= least) {
#pragma unroll
                        for (int j = 0; j < kChunk; j++)
                            if (v[j] >= least) list[atomicAdd(&sh.pending[warp], 1)] = key_of(v[j], (uint32_t)(head + ch * kChunk + j));
                    }
                    __syncwarp();
                    flush(false);
                }
            }
        }
        // the elements outside the aligned words, fewer than 8 + kChunk: one a lane, first block and warp
        if (rank == 0 && warp == 0) {
            const int extra = head + (int)(V - body);
            const int64_t i = lane < head ? lane : body + (lane - head);
            if (lane < extra) {
                const float v = to_f32(x[i]);
                if (v > a.m) a.raise(v, c);
                const float t = max_nan((v - a.m) * c, -200.0f), e = exp2_fast(t);
                a.s += e;
                a.u = fmaf(t, e, a.u);
                // some of these come before all others: an equal logit may win
                if (n_alt > 0 && v >= kLowest) list[atomicAdd(&sh.pending[warp], 1)] = key_of(v, (uint32_t)i);
            }
            __syncwarp();
        }
        if (n_alt > 0) flush(true);
        // warp, block, cluster: always in the same order
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const Sums b{__shfl_xor_sync(0xFFFFFFFFu, a.m, o), __shfl_xor_sync(0xFFFFFFFFu, a.s, o), __shfl_xor_sync(0xFFFFFFFFu, a.u, o)};
            a.add(b, c);
        }
        if (lane == 0) sh.sums[warp] = a;
        sh.best[warp][lane] = mine;
        __syncthreads();
        if (warp == 0) {
            a = sh.sums[0];
            for (int w = 1; w < kWarps; w++) a.add(sh.sums[w], c);
            if (n_alt > 0)
                for (int w = 1; w < kWarps; w++) mine = merge32(mine, sh.best[w][lane], lane);
            if (splits > 1) {
                sh.best[0][lane] = mine;
                if (lane == 0) sh.block_sums = a;
            }
        }
        if (splits > 1) {
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            if (rank == 0 && warp == 0) {
                const uint32_t sums_at = (uint32_t)__cvta_generic_to_shared(&sh.block_sums), best_at = (uint32_t)__cvta_generic_to_shared(&sh.best[0][lane]);
                for (int p = 1; p < splits; p++) {
                    uint32_t at;
                    Sums b;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(sums_at), "r"(p));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.m) : "r"(at) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.s) : "r"(at + 4) : "memory");
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(b.u) : "r"(at + 8) : "memory");
                    a.add(b, c);
                    if (n_alt > 0) {
                        uint64_t k;
                        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(best_at), "r"(p));
                        asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(k) : "r"(at) : "memory");
                        mine = merge32(mine, k, lane);
                    }
                }
            }
        }
        // s: NaN where the row holds a NaN or +inf, 0 where it is masked as a whole
        const float nan = __uint_as_float(0x7FC00000u);
        if (rank == 0) {
            if (warp == 0) {
                const bool bad = a.s != a.s, empty = a.s == 0.0f;
                const float log_s = empty ? 0.0f : logf(a.s), m = bad ? nan : (empty ? 0.0f : a.m);
                if (lane == 0) {
                    sh.stats[0] = m;
                    sh.stats[1] = log_s;
                    if (entropy != nullptr) entropy[row] = bad ? nan : (empty ? 0.0f : log_s - kLn2 * (a.u / a.s));
                }
                if (lane < n_alt) {
                    const uint32_t o = (uint32_t)(mine >> 32);
                    const bool none = bad || mine == 0ull;
                    alts[row * n_alt + lane] = none ? -1 : (int32_t)~(uint32_t)mine;
                    alt_logprobs[row * n_alt + lane] = bad ? nan : (none ? -INFINITY : (value_of(o) - m) * scale - log_s);
                }
            }
            __syncthreads();
            for (int g = threadIdx.x; g < n_given; g += kThreads) {
                const int32_t tok = tokens[row * n_given + g];
                logprobs[row * n_given + g] = tok >= 0 && tok < V ? (to_f32(x[tok]) - sh.stats[0]) * scale - sh.stats[1] : -INFINITY;
            }
        }
        // nobody's lists go away (or are overwritten by the next row) while they are read
        if (splits > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        else __syncthreads();
    }
}

template <int DT>
int launch(const void* logits, int64_t t, int64_t v, int64_t row_stride, float scale, const int32_t* tokens, int n_given, float* logprobs, float* entropy,
           int n_alt, int32_t* alts, float* alt_logprobs, cudaStream_t stream) {
    using T = typename Elem<DT>::T;
    int dev = 0, sms = 0;
    DSX_CUDA(cudaGetDevice(&dev));
    DSX_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // few rows: as many blocks a row as still give every thread two chunks, and no more than two blocks an SM in all
    int splits = 1;
    while (splits < kMaxCluster && t * splits * 2 <= 2 * sms && v >= (int64_t)splits * 2 * 2 * kThreads * Chunk<T>::n) splits *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(t, splits > 1 ? t : (int64_t)1 << 30) * splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = n_alt > 0 ? sizeof(uint64_t) * kWarps * (64 + 32 * Chunk<T>::n) : 0;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 1 : 0;
    DSX_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<DT>, logits, t, v, row_stride, scale, tokens, n_given, logprobs, entropy, n_alt, alts, alt_logprobs,
                                splits));
    DSX_LAUNCHED();
    return DSX_OK;
}

}  // namespace
}  // namespace dsx

using namespace dsx;

extern "C" int dsx_token_logprobs(const void* logits, int dtype, int64_t t, int64_t v, int64_t row_stride, float inv_temperature, const int32_t* tokens,
                                  int n_given, float* logprobs, float* entropy, int n_alt, int32_t* alts, float* alt_logprobs, dsx_stream_t stream) {
    DSX_REQUIRE(dtype_ok(dtype), "token_logprobs: unknown element type %d", dtype);
    DSX_REQUIRE(t >= 0 && t <= 0x0FFFFFFF && v >= 1 && v <= 0x7FFFFFFF, "token_logprobs: %lld rows of %lld logits", (long long)t, (long long)v);
    DSX_REQUIRE(n_given >= 0 && n_given <= 1024 && n_alt >= 0 && n_alt <= kMaxAlt, "token_logprobs: %d given tokens (at most 1024), %d alternatives (at most 32)",
                n_given, n_alt);
    DSX_REQUIRE(inv_temperature >= 1.0e-6f && inv_temperature <= 1.0e6f, "token_logprobs: inverse temperature %g (1e-6 to 1e6)", inv_temperature);
    if (t == 0) return DSX_OK;
    DSX_REQUIRE(row_stride >= v || t == 1, "token_logprobs: row stride %lld below the %lld logits of a row", (long long)row_stride, (long long)v);
    DSX_REQUIRE(logits && (n_given == 0 || (tokens && logprobs)) && (n_alt == 0 || (alts && alt_logprobs)), "token_logprobs: null argument");
    DSX_REQUIRE(((uintptr_t)logits & (dtype_size(dtype) - 1)) == 0, "token_logprobs: logits must be aligned to their elements");
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT) return launch<DT>(logits, t, v, row_stride, inv_temperature, tokens, n_given, logprobs, entropy, n_alt, alts, alt_logprobs, s)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    DSX_GO(DSX_F16);
#undef DSX_GO
}
