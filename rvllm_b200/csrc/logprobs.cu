// Log probabilities of given tokens: for every row x of logits and its token t
//   log p_t = x_t - log sum_j exp(x_j),  rank = 1 + #{j : x_j > x_t},  H = -sum_j p_j log p_j,
// and the `top` largest x_j (equal ones in the order of j) with their log probabilities.
//
// The row is read once.  A thread keeps its largest x so far, m, and s = sum 2^u, w = sum 2^u u with
// u = (x - m) log2(e); an m that moves by d (in units of log2) makes s' = s 2^d, w' = (w + s d) 2^d.  Then
// log p = (x - m) - log s and H = log s - ln 2 w / s.  x - m comes first, so logits of a type's lowest value are
// ordinary numbers.
//
// The largest: a warp keeps the best 32 so far, sorted over its lanes, as 64-bit keys (the value's bits in the order of
// values, then the index reversed), so one comparison has both.  Values above the last one wanted collect in a
// buffer of shared memory and are sorted and merged 32 at a time (bitonic); while the list is not full yet the
// 32 lanes' largest give a first bound, and the block's warps share their bounds, so few values get that far.
//
// A row is a cluster's of 1 to 8 blocks (as many as the GPU has room for when rows are few); parts meet in the
// first block's shared memory in a fixed order, so a row's results do not depend on what else is in the launch.
// Bound by reading the logits.
#include "common.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_MAX_CLUSTER 8
#define LP_LOG2E 1.4426950408889634f
#define LP_LN2 0.6931471805599453f

typedef unsigned long long u64;

__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {       // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
// Larger values have larger keys; NaN and places without a value: 0.  (x + 0: both zeros are equal.)
__device__ __forceinline__ unsigned lp_key(float x) {
    const unsigned b = __float_as_uint(x + 0.f);
    return x != x ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float lp_value(unsigned k) {
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ u64 lp_exchange(u64 x, int mask, bool larger) {
    const u64 y = __shfl_xor_sync(0xffffffffu, x, mask);
    return (x > y) == larger ? x : y;
}
// Descending over the lanes.
__device__ __forceinline__ u64 lp_sort(u64 x, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) x = lp_exchange(x, j, ((lane & j) == 0) == ((lane & k) == 0));
    return x;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ u64 lp_merge(u64 a, u64 b, int lane) {
    const u64 r = __shfl_sync(0xffffffffu, b, 31 - lane);
    u64 x = a > r ? a : r;
#pragma unroll
    for (int j = 16; j > 0; j >>= 1) x = lp_exchange(x, j, (lane & j) == 0);
    return x;
}

template <typename T> struct LpVec;
template <> struct LpVec<float> {
    static constexpr int N = 4, UNROLL = 4;
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const float4 f = __ldcs((const float4*)p);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8, UNROLL = 2;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* v) {
        const uint4 u = __ldcs((const uint4*)p);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
};

struct LpPart { float m, s, w; int above; };

// What a part leaves for the row's first block.
struct LpShared {
    LpPart part[LP_WARPS];
    LpPart whole;
    u64 list[LP_WARPS][32];
    u64 buffer[LP_WARPS][64];
    unsigned bound;
};

__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void lp_add(LpPart& a, float m, float s, float w) {
    // both to the larger reference
    const float top = fmaxf(a.m, m), c = lp_ref(top);
    if (a.s != 0.f) {
        const float d = (lp_ref(a.m) - c) * LP_LOG2E, f = lp_exp2(d);
        a.w = (a.w + a.s * d) * f;
        a.s *= f;
    }
    if (s != 0.f) {
        const float d = (lp_ref(m) - c) * LP_LOG2E, f = lp_exp2(d);
        a.w += (w + s * d) * f;
        a.s += s * f;
    }
    a.m = top;
}

template <typename T, bool TOP>
struct LpThread {
    static constexpr int N = LpVec<T>::N, U = LpVec<T>::UNROLL, E = N * U;
    float m = -INFINITY, s = 0.f, w = 0.f;
    int above = 0;
    float given;
    u64 best = 0;                      // this lane's place of the warp's list
    u64 last = 0;                      // the list's last wanted key
    int waiting = 0;                   // values in the buffer
    int top, lane;
    LpShared& sh;
    u64* buffer;

    __device__ __forceinline__ LpThread(LpShared& shared, int k, float x)
        : given(x), top(k), lane(threadIdx.x & 31), sh(shared), buffer(shared.buffer[threadIdx.x >> 5]) {}

    __device__ __forceinline__ void flush() {            // the first 32 of the buffer into the list
        __syncwarp();
        const u64 x = lane < waiting ? buffer[lane] : 0ull;
        best = lp_merge(best, lp_sort(x, lane), lane);
        last = __shfl_sync(0xffffffffu, best, top - 1);
        if (lane == 0) atomicMax(&sh.bound, (unsigned)(last >> 32));
        __syncwarp();
        if (lane + 32 < waiting) buffer[lane] = buffer[lane + 32];
        waiting = max(0, waiting - 32);
        __syncwarp();
    }
    // E values of this thread (every lane of the warp comes here): x[i] is column col(i); `real(i)`: it exists.
    template <typename Col, typename Real>
    __device__ __forceinline__ void take(const float (&x)[E], Col col, Real real) {
        float bm = x[0];
#pragma unroll
        for (int i = 1; i < E; ++i) bm = fmaxf(bm, x[i]);
        if (bm > m) {
            if (s != 0.f) {
                const float d = (m - bm) * LP_LOG2E, f = lp_exp2(d);
                w = (w + s * d) * f;
                s *= f;
            }
            m = bm;
        }
        const float c = lp_ref(m);
        float s2[2] = {0.f, 0.f}, w2[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            // (far below: 2^t is 0, and so is its product with t)
            const float t = lp_max_nan((x[i] - c) * LP_LOG2E, -200.f), e = lp_exp2(t);
            s2[i & 1] += e;
            w2[i & 1] = fmaf(e, t, w2[i & 1]);
            above += x[i] > given;
        }
        s += s2[0] + s2[1];
        w += w2[0] + w2[1];
        if (TOP) {
            const unsigned own = (unsigned)(last >> 32);
            unsigned shared = *(volatile unsigned*)&sh.bound;
            const unsigned mine = bm == bm ? lp_key(bm) : 0u;
            if (!__any_sync(0xffffffffu, mine >= own && mine >= shared)) return;
            if (last == 0ull) {
                // no full list yet: as many values as are wanted reach the lanes' largest down to this one
                const u64 sorted = lp_sort((u64)mine << 32, lane);
                shared = max(shared, (unsigned)(__shfl_sync(0xffffffffu, sorted, top - 1) >> 32));
            }
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const unsigned k = real(i) ? lp_key(x[i]) : 0u;
                const u64 whole = ((u64)k << 32) | (0xffffffffu - (unsigned)col(i));
                const bool in = k != 0u && whole > last && k >= shared;
                const unsigned who = __ballot_sync(0xffffffffu, in);
                if (who) {
                    if (in) buffer[waiting + __popc(who & ((1u << lane) - 1u))] = whole;
                    waiting += __popc(who);
                    if (waiting >= 32) flush();
                }
            }
        }
    }
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_kernel(
    const T* __restrict__ logits, long long row_stride, int vocab, const int* __restrict__ tokens, int top,
    float* __restrict__ logprob, int* __restrict__ rank, float* __restrict__ entropy, float* __restrict__ top_logprob,
    int* __restrict__ top_id, int parts) {
    rv_pdl_prologue();
    constexpr int N = LpVec<T>::N, U = LpVec<T>::UNROLL, E = N * U;
    __shared__ LpShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - row * parts);
    const T* x = logits + row * row_stride;
    const int token = tokens[row];
    const bool known = token >= 0 && token < vocab;
    const float given = known ? rv_load(x + token) : INFINITY;
    if (tid == 0) sh.bound = 0u;
    __syncthreads();
    LpThread<T, TOP> th(sh, top, given);
    // whole 16-byte vectors from the first aligned one on, shared out over the parts; what lies
    // before and behind them is the last part's
    const int head = min(vocab, (int)((((16 - ((uintptr_t)x & 15)) & 15)) / sizeof(T)));
    const int vectors = (vocab - head) / N, tail = head + vectors * N;
    const int v0 = (int)((long long)vectors * part / parts), v1 = (int)((long long)vectors * (part + 1) / parts);
    const T* body = x + head;
    float v[E];
    int at = v0;
    for (; at + U * LP_THREADS <= v1; at += U * LP_THREADS) {
#pragma unroll
        for (int u = 0; u < U; ++u) LpVec<T>::load(body + (size_t)(at + u * LP_THREADS + tid) * N, v + u * N);
        const int base = head + (at + tid) * N;
        th.take(v, [&](int i) { return base + (i / N) * LP_THREADS * N + i % N; }, [](int) { return true; });
    }
    if (at < v1) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at + u * LP_THREADS + tid < v1) {
                LpVec<T>::load(body + (size_t)(at + u * LP_THREADS + tid) * N, v + u * N);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i) v[u * N + i] = -INFINITY;
            }
        }
        const int base = head + (at + tid) * N;
        th.take(v, [&](int i) { return base + (i / N) * LP_THREADS * N + i % N; },
                [&](int i) { return at + (i / N) * LP_THREADS + tid < v1; });
    }
    if (part == parts - 1 && warp == 0 && head + vocab - tail > 0) {
        const int col = lane < head ? lane : tail + lane - head;
        const bool have = col < vocab;
        v[0] = have ? rv_load(x + col) : -INFINITY;
#pragma unroll
        for (int i = 1; i < E; ++i) v[i] = -INFINITY;
        th.take(v, [&](int) { return col; }, [&](int i) { return i == 0 && have; });
    }
    if (TOP) {
        while (th.waiting > 0) th.flush();
        sh.list[warp][lane] = th.best;
    }
    // ---- the warp's, the block's, the cluster's ------------------------------------------------
    {
        const float most = rv_warp_max(th.m), c = lp_ref(most);
        float s = 0.f, w = 0.f;
        if (th.s != 0.f) {
            const float d = (lp_ref(th.m) - c) * LP_LOG2E, f = lp_exp2(d);
            s = th.s * f;
            w = (th.w + th.s * d) * f;
        }
        s = rv_warp_sum(s);
        w = rv_warp_sum(w);
        const int above = __reduce_add_sync(0xffffffffu, th.above);
        if (lane == 0) sh.part[warp] = {most, s, w, above};
    }
    __syncthreads();
    if (tid == 0) {
        LpPart p = sh.part[0];
        for (int i = 1; i < LP_WARPS; ++i) {
            lp_add(p, sh.part[i].m, sh.part[i].s, sh.part[i].w);
            p.above += sh.part[i].above;
        }
        sh.whole = p;
    }
    if (TOP) {
#pragma unroll
        for (int step = LP_WARPS / 2; step > 0; step >>= 1) {
            if (warp < step) {
                th.best = lp_merge(th.best, sh.list[warp + step][lane], lane);
                sh.list[warp][lane] = th.best;
            }
            __syncthreads();
        }
    }
    if (parts > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (part == 0 && warp == 0) {
            auto remote = [](const void* p, int rank_) {
                unsigned a;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank_));
                return a;
            };
            LpPart p = sh.whole, q[LP_MAX_CLUSTER];
            u64 lists[LP_MAX_CLUSTER];
#pragma unroll
            for (int k = 1; k < LP_MAX_CLUSTER; ++k)
                if (k < parts) {
                    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(q[k].m), "=f"(q[k].s), "=f"(q[k].w), "=r"(q[k].above) : "r"(remote(&sh.whole, k)) : "memory");
                    if (TOP) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(lists[k]) : "r"(remote(&sh.list[0][lane], k)) : "memory");
                }
#pragma unroll
            for (int k = 1; k < LP_MAX_CLUSTER; ++k)
                if (k < parts) {
                    lp_add(p, q[k].m, q[k].s, q[k].w);
                    p.above += q[k].above;
                    if (TOP) th.best = lp_merge(th.best, lists[k], lane);
                }
            if (lane == 0) sh.whole = p;
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // nobody leaves while it is read
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    if (part != 0 || warp != 0) return;
    __syncwarp();
    const LpPart p = sh.whole;
    const float c = lp_ref(p.m), logs = logf(p.s);
    if (lane == 0) {
        const float h = logs - LP_LN2 * (p.w / p.s);
        logprob[row] = known ? (given - c) - logs : NAN;
        rank[row] = known ? p.above + 1 : 0;
        entropy[row] = h < 0.f ? 0.f : h;
    }
    if (TOP && lane < top) {
        const bool have = th.best != 0ull;
        const float y = lp_value((unsigned)(th.best >> 32));
        top_logprob[row * top + lane] = have ? (y - c) - logs : NAN;
        top_id[row * top + lane] = have ? (int)(0xffffffffu - (unsigned)th.best) : -1;
    }
}

extern "C" int rv_token_logprobs(const void* logits, int dtype, long long row_stride, int rows, int vocab, const int* tokens,
                                 int top, float* logprob, int* rank, float* entropy, float* top_logprob, int* top_id,
                                 void* stream) {
    if (rows == 0) return 0;
    if (rows < 0 || vocab <= 0) RV_FAIL("token_logprobs: bad sizes");
    if (top < 0 || top > 32 || top > vocab) RV_FAIL("token_logprobs: %d alternatives (0 to 32, at most the vocabulary)", top);
    // blocks a row: until there are some two a multiprocessor, parts of four rounds of loads at least
    const int size = dtype == RV_DTYPE_F32 ? 4 : 2, sms = rv_sm_count();
    int parts = 1;
    while (2 * parts <= LP_MAX_CLUSTER && (long long)rows * 2 * parts <= 4ll * sms &&
           (long long)vocab * size >= (long long)2 * parts * LP_THREADS * 16)
        parts *= 2;
    if ((long long)rows * parts > 0x7fffffffLL) RV_FAIL("token_logprobs: too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * parts);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = rv_pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = parts > 1 ? 2 : 1;
    cudaError_t e = cudaSuccess;
    RV_DISPATCH_DTYPE(dtype, "token_logprobs",
                      auto kernel = top ? token_logprobs_kernel<T, true> : token_logprobs_kernel<T, false>;
                      e = cudaLaunchKernelEx(&cfg, kernel, (const T*)logits, row_stride, vocab, tokens, top, logprob, rank, entropy,
                                             top_logprob, top_id, parts));
    if (e != cudaSuccess) RV_FAIL("token_logprobs: %s", cudaGetErrorString(e));
    RV_CHECK_LAUNCH("token_logprobs");
    return 0;
}
