// Log probabilities of given tokens, entropy and the most likely alternatives, from rows of logits, in one pass over them.
//
// With z = logit * scale, m the row's largest logit, d = (logit - m) * scale:   s = sum e^d,   u = sum d e^d,
//   log p(token) = d(token) - ln s,   entropy = ln s - u / s,   alternatives = the n_alt largest logits (equal logits: lower index).
// Counterparts in the reference (paths relative to the deepstrix repository): its sampler's softmax over the vocabulary
// (crates/v4flash-kernels/kernels/softmax_sample.hip) and the teacher-forced scoring of tests/v41_golden_gate.rs.
//
// One pass.  A thread keeps its own running maximum and its s and u relative to it; it takes 32 bytes of logits at a time and rescales
// only when their maximum is new.  Pairs of f32 go through the packed add, multiply and fused multiply-add of sm_100: an element costs
// about five and a half issue slots, one of them the exponential.
// The alternatives cost the loop nothing: afterwards the n_alt-th largest of the maxima of 32 or 64 groups of threads is a value that
// at least n_alt logits reach, and hardly more do, so only the threads whose maximum reaches it have their chunks read again (from L2) for
// the few logits that do; those are ranked by counting.  Where more than the list holds reach it -- a row of equal logits, say, or one masked with the
// lowest value -- a second pass keeps the best 32 of every warp in registers, sorting candidates 32 at a time.  That comes on top: every
// logit that reaches the threshold has been counted by then, a shared atomic each.  64 rows of 131072 f32 that hold the lowest value but for three
// logits take 45.5 us with twenty alternatives where random rows take 10.5 (and rows masked by -inf 9.5), 512 such rows 240 and 57.
// A row belongs to one block, or, when there are few rows, to the blocks of a cluster that join their sums and lists through
// distributed shared memory: one launch, no workspace, and the order of every addition is fixed.
//
// Bound: HBM; bf16 and f16 rows at the full rate are 11.6 elements a clock and SM, of which the exponentials can take 16.  2048 rows of 131072
// f32 take 160 us without and 173 with five alternatives, 6.7 and 6.2 TB/s (167 and 180 after a second of it); 4096 of bf16 174 and 187
// (the part behind the loop of one block in five at a time), 200 and 212 once the power cap holds the clock, 5.1 TB/s; 64 rows of f32 with twenty
// 16 us from HBM and 10.5 from L2, one row of 32000 6, latency.  A ring of asynchronous copies that ran on into the next row was
// slower (227 us when the loop took 199: its instructions, not the loads in flight, were what the loop lacked), and so were chunks requested 2 to 6
// ahead for a few rows (0.1 to 1.3 us more), and keeping the chunk of every thread's maximum so that it need not be read again (loop 5 to 10 % longer).
#include "head.cuh"

namespace dsx {
namespace {

constexpr int kMaxAlt = 32;            // one per lane of the warp that holds a list
constexpr int kMaxCluster = 8;
constexpr int kMaxGiven = 1024, kFetched = 64;   // given tokens of a row; of which are fetched ahead
constexpr float kLowest = -3.402823466e38f;
constexpr uint32_t kFloor = 0x00800000u;   // order_of(kLowest): nothing finite is below it
constexpr float kLn2 = 0.6931471805599453f, kLog2e = 1.4426950408889634f;

// 2^x; the instruction is off by at most 2 ulp, and 0 for x below -126 (subnormal results are flushed)
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

__device__ __forceinline__ void cluster_sync_all() {
    __syncwarp();   // the .aligned forms want the warp together, whatever branch came before
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// where the first block of the cluster has `p`
__device__ __forceinline__ uint32_t in_first_block(const void* p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)));
    return r;
}

// 32 bytes of logits: 8 floats or 16 halves, as they were loaded.
template <typename T> struct Chunk;
template <> struct Chunk<float> {
    static constexpr int n = 8;
    __device__ static void two(const uint32_t (&w)[8], int j, float& a, float& b) { a = __uint_as_float(w[2 * j]); b = __uint_as_float(w[2 * j + 1]); }
    __device__ static float top(const uint32_t (&w)[8]) {
        float t = __uint_as_float(w[0]);
#pragma unroll
        for (int j = 1; j < 8; j++) t = fmaxf(t, __uint_as_float(w[j]));
        return t;
    }
};
template <typename T> struct HalfChunk {
    static constexpr int n = 16;
    __device__ static void two(const uint32_t (&w)[8], int j, float& a, float& b) { const float2 f = unpack2<T>(w[j]); a = f.x; b = f.y; }
};
template <> struct Chunk<__nv_bfloat16> : HalfChunk<__nv_bfloat16> {
    __device__ static float top(const uint32_t (&w)[8]) {
        __nv_bfloat162 t = *reinterpret_cast<const __nv_bfloat162*>(&w[0]);
#pragma unroll
        for (int j = 1; j < 8; j++) t = __hmax2(t, *reinterpret_cast<const __nv_bfloat162*>(&w[j]));
        return fmaxf(__low2float(t), __high2float(t));
    }
};
template <> struct Chunk<__half> : HalfChunk<__half> {
    __device__ static float top(const uint32_t (&w)[8]) {
        __half2 t = *reinterpret_cast<const __half2*>(&w[0]);
#pragma unroll
        for (int j = 1; j < 8; j++) t = __hmax2(t, *reinterpret_cast<const __half2*>(&w[j]));
        return fmaxf(__low2float(t), __high2float(t));
    }
};
template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, uint32_t (&w)[8]) {
    const uint4 w0 = __ldg(reinterpret_cast<const uint4*>(p)), w1 = __ldg(reinterpret_cast<const uint4*>(p) + 1);
    w[0] = w0.x; w[1] = w0.y; w[2] = w0.z; w[3] = w0.w; w[4] = w1.x; w[5] = w1.y; w[6] = w1.z; w[7] = w1.w;
}

// A thread's sums relative to its maximum: of 2^t and of t 2^t with t = (x - m) * c.  s = 0 exactly where nothing has been seen.
struct Sums {
    float m, s, u;
    // to a maximum at least as large; s = 0 stays 0 whatever the difference
    __device__ __forceinline__ void raise(float to, float c) {
        const float t = fmaxf((m - to) * c, -200.0f), e = exp2_fast(t);
        u = (u + s * t) * e;
        s *= e;
        m = to;
    }
};

constexpr int kList = 512;   // candidates the block ranks by counting

template <int NT>
struct alignas(16) Shared {
    static constexpr int kWarps = NT / 32;
    alignas(16) uint32_t group_top[64];     // order of the maxima of 32 or 64 groups of threads, 0 where they saw nothing
    float warp_m[kWarps], warp_s[kWarps], warp_u[kWarps];
    int n_readers;                          // threads whose maximum reaches the threshold,
    int reader[NT];                         // in any order
    int count;                              // candidates that reach it
    uint64_t warp_list[kWarps][96];         // second pass: a warp's candidates, at most 31 left over and two of every lane
    alignas(16) uint64_t list[kList + 2];
    alignas(16) uint64_t cluster_list[NT == 64 ? 2 : kMaxCluster * kMaxAlt];   // first block of a cluster: the bests of all blocks,
    float sums[kMaxCluster][3];                                 // and their sums
    uint64_t best[kMaxAlt];                 // the part's best, descending, 0 = nothing
    float given[kFetched];                  // logits of the first given tokens
    bool outside[kFetched];                 // no such token
};

// best[0 .. n_alt) = the n_alt largest of the n keys of `list`, descending: a key's place is the number of larger ones (keys are
// distinct but for 0, "nothing", which takes no place).  Keys are read two at a time; what lies behind an odd end is not counted.
template <int NT>
__device__ __forceinline__ void rank_list(const uint64_t* list, int n, int n_alt, uint64_t* best) {
    for (int i = threadIdx.x; i < n; i += NT) {
        const uint64_t k = list[i];
        int r = 0;
        for (int j = 0; j < n; j += 2) {
            const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(list + j);
            r += (o.x > k ? 1 : 0) + (o.y > k && j + 1 < n ? 1 : 0);
        }
        if (k != 0ull && r < n_alt) best[r] = k;
    }
}

// NT threads a block: 256, or 64 for many short rows, whose time is the part behind the loop.  48 registers a thread (1280 threads an SM, 40 KB
// of logits in flight) against 64 (1024 threads): 4096 rows of 131072 bf16 191 us against 198, 2048 of f32 172 against 191.  The f16 kernels
// spill 20 and 32 bytes at 48 registers, the others nothing.
template <int DT, int NT>
__global__ void __launch_bounds__(NT, 1280 / NT)
token_logprobs_kernel(const void* __restrict__ logits, int64_t V, int64_t row_stride, float scale, const int32_t* __restrict__ tokens, int n_given,
                      float* __restrict__ logprobs, float* __restrict__ entropy, int n_alt, int32_t* __restrict__ alts, float* __restrict__ alt_logprobs,
                      int splits) {
    using T = typename Elem<DT>::T;
    using Ch = Chunk<T>;
    constexpr int kChunk = Ch::n;
    constexpr int kThreads = NT, kWarps = NT / 32;
    __shared__ Shared<NT> sh;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = splits > 1 ? (int)(blockIdx.x % (unsigned)splits) : 0;
    const int64_t row = blockIdx.x / (unsigned)splits;
    const float c = scale * kLog2e;
    const T* __restrict__ x = reinterpret_cast<const T*>(logits) + row * row_stride;
    if (threadIdx.x < 64) sh.group_top[threadIdx.x] = 0u;
    if (threadIdx.x < kMaxAlt) sh.best[threadIdx.x] = 0ull;
    if (threadIdx.x == 0) {
        sh.count = 0;
        sh.n_readers = 0;
    }
    __syncthreads();
    if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this block has started; waited for behind the loop
    pdl_wait();   // the logits may come from the kernel before this one
    // whole 16-byte words from the row's first aligned element on; the few elements before and after them one by one
    const int head = (int)min((int64_t)(((16u - (uint32_t)((uintptr_t)x & 15u)) & 15u) / sizeof(T)), V);
    const uint32_t n_chunks = (uint32_t)((V - head) / kChunk);   // below 2^28
    const int64_t body = head + (int64_t)n_chunks * kChunk;
    const int extra = rank == 0 ? head + (int)(V - body) : 0;          // fewer than 8 + kChunk, one a lane of the first block's first warp
    const uint32_t extra_at = lane < head ? (uint32_t)lane : (uint32_t)body + (uint32_t)(lane - head);
    const bool has_extra = warp == 0 && lane < extra;
    // chunk i of this thread is first + i * step
    const uint32_t step = (uint32_t)(kThreads * splits), part = (uint32_t)(rank * kThreads), first = part + threadIdx.x;
    const T* chunks = x + head;

    // ------------------------------------------------------------------ sums
    Sums a{kLowest, 0.0f, 0.0f};
    if (has_extra) {
        const float v = to_f32(x[extra_at]);
        if (v > a.m) a.m = v;
        const float t = max_nan((v - a.m) * c, -200.0f);
        a.s = exp2_fast(t);
        a.u = t * a.s;
    }
    {
        uint64_t s2 = pair(a.s, 0.0f), u2 = pair(a.u, 0.0f);
        const uint64_t c2 = pair(c, c);
        uint32_t next[8];
        if (first < n_chunks) load_chunk(chunks + (int64_t)first * kChunk, next);
        if (rank == 0)   // two dependent loads that the first chunk's latency covers
            for (int g = threadIdx.x; g < min(n_given, kFetched); g += kThreads) {
                const int32_t tok = tokens[row * n_given + g];
                const bool in = tok >= 0 && tok < V;
                sh.given[g] = in ? to_f32(x[tok]) : 0.0f;
                sh.outside[g] = !in;
            }
        for (uint32_t ch = first; ch < n_chunks; ch += step) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = next[j];
            if (ch + step < n_chunks) load_chunk(chunks + (int64_t)(ch + step) * kChunk, next);   // requested before this one's work
            const float top = Ch::top(w);
            if (top > a.m) {
                const float t = fmaxf((a.m - top) * c, -200.0f), e = exp2_fast(t);
                const uint64_t e2 = pair(e, e);
                u2 = mul2(fma2(s2, pair(t, t), u2), e2);
                s2 = mul2(s2, e2);
                a.m = top;
            }
            const uint64_t minus_m = pair(-a.m, -a.m);
#pragma unroll
            for (int j = 0; j < kChunk / 2; j++) {
                float v0, v1, t0, t1;
                Ch::two(w, j, v0, v1);
                unpair(mul2(add2(pair(v0, v1), minus_m), c2), t0, t1);
                t0 = max_nan(t0, -200.0f);     // a masked logit: 2^-200 is 0, and 0 * -200 too
                t1 = max_nan(t1, -200.0f);
                const uint64_t e = pair(exp2_fast(t0), exp2_fast(t1));
                s2 = add2(s2, e);
                u2 = fma2(pair(t0, t1), e, u2);
            }
        }
        float s0, s1, u0, u1;
        unpair(s2, s0, s1);
        unpair(u2, u0, u1);
        a.s = s0 + s1;
        a.u = u0 + u1;
    }

    // A warp's sums, and the maxima of 32 groups of threads, or of 64 for many alternatives (a threshold that is the least of few maxima lets
    // more than four times as many candidates through: 64 rows of 131072 with 32 alternatives 13 us, 21 with 32 groups).  All sums are added in an order that does not depend on timing.
    const bool many = n_alt > 16;
    __syncwarp();
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every block of the cluster has started
    {
        float m = a.m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        if (n_alt > 0 && a.s != 0.0f) atomicMax(&sh.group_top[threadIdx.x & (many ? 63 : 31)], order_of(a.m));
        Sums r = a;
        r.raise(m, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            r.s += __shfl_xor_sync(0xFFFFFFFFu, r.s, o);
            r.u += __shfl_xor_sync(0xFFFFFFFFu, r.u, o);
        }
        if (lane == 0) {
            sh.warp_m[warp] = m;
            sh.warp_s[warp] = r.s;
            sh.warp_u[warp] = r.u;
        }
    }
    __syncthreads();
    if (warp == kWarps - 1) {   // the part's sums, to the row's first block
        Sums p{kLowest, 0.0f, 0.0f};
        if (lane < kWarps) p = Sums{sh.warp_m[lane], sh.warp_s[lane], sh.warp_u[lane]};
        float m = p.m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        p.raise(m, c);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            p.s += __shfl_xor_sync(0xFFFFFFFFu, p.s, o);
            p.u += __shfl_xor_sync(0xFFFFFFFFu, p.u, o);
        }
        const float v = lane == 0 ? m : (lane == 1 ? p.s : p.u);
        if (lane < 3) {
            if (splits > 1) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(in_first_block(&sh.sums[rank][lane])), "f"(v) : "memory");
            else sh.sums[0][lane] = v;
        }
        __syncwarp();
    }

    // ---------------------------------------------------------- alternatives
    if (n_alt > 0) {
        // the n_alt-th largest of the groups' maxima = the smallest that fewer than n_alt of them are above: n_alt logits reach it
        auto reached = [&](uint32_t mine, int groups) {
            int above = 0;
#pragma unroll 8
            for (int j = 0; j < groups / 4; j++) {
                const uint4 o = reinterpret_cast<const uint4*>(sh.group_top)[j];
                above += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
            }
            return above < n_alt ? mine : 0xFFFFFFFFu;
        };
        uint32_t reach = reached(sh.group_top[lane], many ? 64 : 32);
        if (many) reach = min(reach, reached(sh.group_top[lane + 32], 64));
        const uint32_t threshold = max(__reduce_min_sync(0xFFFFFFFFu, reach), kFloor);
        const float least = value_of(threshold);
        auto push = [&](float v, uint32_t i) {
            const int at = atomicAdd(&sh.count, 1);
            if (at < kList) sh.list[at] = key_of(v, i);
        };
        if (has_extra) {
            const float v = to_f32(x[extra_at]);
            if (v >= least) push(v, (uint32_t)extra_at);
        }
        const bool reaches = a.s != 0.0f && a.m >= least;
        const uint32_t again = __ballot_sync(0xFFFFFFFFu, reaches);
        if (again) {
            int place = 0;
            if (lane == 0) place = atomicAdd(&sh.n_readers, __popc(again));
            place = __shfl_sync(0xFFFFFFFFu, place, 0);
            if (reaches) sh.reader[place + __popc(again & ((1u << lane) - 1u))] = (int)threadIdx.x;
        }
        __syncthreads();
        // their chunks, shared out over the block: round r of reader i is item i * rounds + r
        const uint32_t rounds = n_chunks > part ? (n_chunks - part + step - 1) / step : 0u, items = (uint32_t)sh.n_readers * rounds;
        for (uint32_t item = threadIdx.x; item < items; item += kThreads) {
            const uint32_t i = item / rounds;
            const uint32_t ch = part + (uint32_t)sh.reader[i] + (item - i * rounds) * step;
            if (ch >= n_chunks) continue;
            uint32_t w[8];
            load_chunk(chunks + (int64_t)ch * kChunk, w);
            if (Ch::top(w) >= least) {
#pragma unroll
                for (int j = 0; j < kChunk / 2; j++) {
                    float v0, v1;
                    Ch::two(w, j, v0, v1);
                    if (v0 >= least) push(v0, head + ch * (uint32_t)kChunk + 2 * j);
                    if (v1 >= least) push(v1, head + ch * (uint32_t)kChunk + 2 * j + 1);
                }
            }
        }
        __syncthreads();
        if (sh.count <= kList) {
            rank_list<NT>(sh.list, sh.count, n_alt, sh.best);
        } else {
            // too many: a second pass over the part, in which a warp keeps its best 32 (one a lane) and lists only what may enter them.
            // Its chunks come in ascending order, so an equal logit behind a full list is out: in this pass, equal logits cost one compare each.
            uint64_t* list = sh.warp_list[warp];
            uint64_t mine = 0ull;
            uint32_t kth = 0u, own = threshold;   // order of the list's n_alt-th; the lowest order that may still enter it
            int pending = 0;   // on the list; the same in every lane, advanced by ballots: no lane can see another count than its neighbours
            auto append = [&](bool in, float v, uint32_t i) {
                const uint32_t who = __ballot_sync(0xFFFFFFFFu, in);
                if (in) list[pending + __popc(who & ((1u << lane) - 1u))] = key_of(v, i);
                pending += __popc(who);
            };
            auto flush = [&](int keep) {   // merge candidates 32 at a time until at most `keep` are left (the last ones padded with nothing)
                if (pending <= keep) return;
                __syncwarp();   // the list is written
                while (pending > keep) {
                    const int n = min(pending, 32);
                    const uint64_t k = lane < n ? list[pending - n + lane] : 0ull;
                    pending -= n;
                    mine = merge32(mine, sort32(k, lane), lane);
                }
                kth = (uint32_t)(__shfl_sync(0xFFFFFFFFu, mine, n_alt - 1) >> 32);
                __syncwarp();   // and read, before it is written again
            };
            for (uint32_t ch = first; ch - lane < n_chunks; ch += step) {
                uint32_t w[8];
                const bool live = ch < n_chunks;
                if (live) load_chunk(chunks + (int64_t)ch * kChunk, w);
                const float least = value_of(own);
                const bool any = live && Ch::top(w) >= least;
                if (__any_sync(0xFFFFFFFFu, any)) {
#pragma unroll 1
                    for (int j = 0; j < kChunk / 2; j++) {
                        float v0 = -INFINITY, v1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < kChunk / 2; i++)
                            if (i == j && any) Ch::two(w, i, v0, v1);
                        const float bar = value_of(max(own, kth));   // within a round an equal logit may have the lower index
                        append(v0 >= bar, v0, head + ch * (uint32_t)kChunk + 2 * j);
                        append(v1 >= bar, v1, head + ch * (uint32_t)kChunk + 2 * j + 1);
                        flush(31);
                    }
                    own = max(own, kth + 1u);
                }
            }
            {   // some of these come before all others: an equal logit may win
                const float v = has_extra ? to_f32(x[extra_at]) : -INFINITY;
                append(v >= kLowest, v, (uint32_t)extra_at);
            }
            flush(0);
            __syncthreads();
            sh.list[threadIdx.x] = mine;   // 256 of them
            __syncthreads();
            rank_list<NT>(sh.list, kThreads, n_alt, sh.best);
        }
    }
    __syncthreads();

    // --------------------------------------------------------------- the row
    if (splits > 1) {
        if (warp == 0 && lane < n_alt)
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(in_first_block(&sh.cluster_list[rank * n_alt + lane])), "l"(sh.best[lane]) : "memory");
        cluster_sync_all();   // nothing is read from or written to another block behind it
        if (rank != 0) return;
        if (n_alt > 0) {
            rank_list<NT>(sh.cluster_list, splits * n_alt, n_alt, sh.best);
            __syncthreads();
        }
    }
    if (warp == 0) {
        Sums p{kLowest, 0.0f, 0.0f};   // a lane per part
        if (lane < splits) p = Sums{sh.sums[lane][0], sh.sums[lane][1], sh.sums[lane][2]};
        float m = p.m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        p.raise(m, c);
        float s = p.s, u = p.u;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
        }
        // s: NaN where the row holds a NaN or +inf, 0 where it is masked as a whole
        const float nan = __uint_as_float(0x7FC00000u);
        const bool bad = s != s, empty = s == 0.0f;
        const float log_s = empty ? 0.0f : logf(s);
        m = bad ? nan : (empty ? 0.0f : m);
        if (lane == 0 && entropy != nullptr) entropy[row] = bad ? nan : (empty ? 0.0f : log_s - kLn2 * (u / s));
        if (lane < n_alt) {
            const uint64_t k = sh.best[lane];
            const bool none = bad || k == 0ull;
            alts[row * n_alt + lane] = none ? -1 : (int32_t)~(uint32_t)k;
            alt_logprobs[row * n_alt + lane] = bad ? nan : (none ? -INFINITY : (value_of((uint32_t)(k >> 32)) - m) * scale - log_s);
        }
        for (int g = lane; g < n_given; g += 32) {
            float v;
            bool in;
            if (g < kFetched) {
                v = sh.given[g];
                in = !sh.outside[g];
            } else {
                const int32_t tok = tokens[row * n_given + g];
                in = tok >= 0 && tok < V;
                v = in ? to_f32(x[tok]) : 0.0f;
            }
            logprobs[row * n_given + g] = in ? (v - m) * scale - log_s : -INFINITY;
        }
    }
}

template <int DT, int NT>
int launch(const void* logits, int64_t t, int64_t v, int64_t row_stride, float scale, const int32_t* tokens, int n_given, float* logprobs, float* entropy,
           int n_alt, int32_t* alts, float* alt_logprobs, int splits, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(t * splits));
    cfg.blockDim = dim3(NT);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = splits > 1 ? 2 : 1;
    DSX_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<DT, NT>, logits, v, row_stride, scale, tokens, n_given, logprobs, entropy, n_alt, alts,
                                alt_logprobs, splits));
    DSX_LAUNCHED();
    return DSX_OK;
}

template <int DT>
int launch_for(const void* logits, int64_t t, int64_t v, int64_t row_stride, float scale, const int32_t* tokens, int n_given, float* logprobs, float* entropy,
               int n_alt, int32_t* alts, float* alt_logprobs, cudaStream_t stream) {
    int sms = 0;
    if (int rc = head_sm_count(&sms)) return rc;
    constexpr int kChunk = Chunk<typename Elem<DT>::T>::n;
    // many rows of at most 16 chunks a thread: the small block (4096 rows of 4096 bf16 15.6 us against 28.4, of 16384 34.2 against 44.7, but
    // of 32000 with 20 alternatives 98 against 72); also a row that a small block reads in one round
    const bool small = v <= 64 * kChunk || (t >= 8 * (int64_t)sms && v <= 16 * 64 * kChunk);
    // few rows: as many blocks a row as still give every thread two chunks, and no more than two blocks an SM in all (64 rows of 131072 f32
    // 20.5 / 14.0 / 11.1 / 13.6 us with 1 / 2 / 4 / 8, 148 of bf16 13.0 / 12.2 / 14.3 / 17.6, one row of 32000 f32 7.0 / 6.6 / 5.8 / 5.4), or as many
    // as are resident where every thread keeps 16 (300 rows of 131072 f32 40.9 / 30.0 / 34.2 us with 1 / 2 / 4, but 333 of 50021 f16 12.7 / 13.6; 250 of
    // 131072 bf16 pay for the rule, 18.5 with two and 17.7 with one)
    int splits = 1;
    auto more = [&](int blocks_per_sm, int chunks) {
        return splits < kMaxCluster && t * splits * 2 <= blocks_per_sm * (int64_t)sms && v >= (int64_t)splits * 2 * chunks * 256 * kChunk;
    };
    while (!small && (more(2, 2) || more(1280 / 256, 16))) splits *= 2;
    if (small) return launch<DT, 64>(logits, t, v, row_stride, scale, tokens, n_given, logprobs, entropy, n_alt, alts, alt_logprobs, splits, stream);
    return launch<DT, 256>(logits, t, v, row_stride, scale, tokens, n_given, logprobs, entropy, n_alt, alts, alt_logprobs, splits, stream);
}

}  // namespace
}  // namespace dsx

using namespace dsx;

extern "C" int dsx_token_logprobs(const void* logits, int dtype, int64_t t, int64_t v, int64_t row_stride, float inv_temperature, const int32_t* tokens,
                                  int n_given, float* logprobs, float* entropy, int n_alt, int32_t* alts, float* alt_logprobs, dsx_stream_t stream) {
    DSX_REQUIRE(dtype_ok(dtype), "token_logprobs: unknown element type %d", dtype);
    DSX_REQUIRE(t >= 0 && t <= 0x0FFFFFFF && v >= 1 && v <= 0x7FFFFFFF, "token_logprobs: %lld rows of %lld logits", (long long)t, (long long)v);
    DSX_REQUIRE(n_given >= 0 && n_given <= kMaxGiven && n_alt >= 0 && n_alt <= kMaxAlt, "token_logprobs: %d given tokens (at most 1024), %d alternatives (at most 32)",
                n_given, n_alt);
    DSX_REQUIRE(inv_temperature >= 1.0e-6f && inv_temperature <= 1.0e6f, "token_logprobs: inverse temperature %g (1e-6 to 1e6)", inv_temperature);
    if (t == 0) return DSX_OK;
    DSX_REQUIRE(row_stride >= v || t == 1, "token_logprobs: row stride %lld below the %lld logits of a row", (long long)row_stride, (long long)v);
    DSX_REQUIRE(logits && (n_given == 0 || (tokens && logprobs)) && (n_alt == 0 || (alts && alt_logprobs)), "token_logprobs: null argument");
    const uintptr_t words = (n_given ? (uintptr_t)tokens | (uintptr_t)logprobs : 0) | (uintptr_t)entropy | (n_alt ? (uintptr_t)alts | (uintptr_t)alt_logprobs : 0);
    DSX_REQUIRE(((uintptr_t)logits & (dtype_size(dtype) - 1)) == 0 && (words & 3) == 0, "token_logprobs: every array must be aligned to its elements");
    const cudaStream_t s = (cudaStream_t)stream;
#define DSX_GO(DT) return launch_for<DT>(logits, t, v, row_stride, inv_temperature, tokens, n_given, logprobs, entropy, n_alt, alts, alt_logprobs, s)
    if (dtype == DSX_F32) DSX_GO(DSX_F32);
    if (dtype == DSX_BF16) DSX_GO(DSX_BF16);
    DSX_GO(DSX_F16);
#undef DSX_GO
}
