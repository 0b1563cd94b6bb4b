// Log probabilities of given tokens: for every row x of logits and its token t
//   log p_t = x_t - log sum_j exp(x_j),  rank = 1 + #{j : x_j > x_t},  H = -sum_j p_j log p_j,
// and the `top` largest x_j (equal ones in the order of j) with their log probabilities.
//
// The row is read once.  A thread keeps its largest x so far, m, and s = sum 2^u, w = sum 2^u u with
// u = (x - m) log2(e); an m that moves by d (in units of log2) makes s' = s 2^d, w' = (w + s d) 2^d.  Then
// log p = (x - m) - log s and H = log s - ln 2 w / s.  x - m comes first, so logits of a type's lowest value are
// ordinary numbers.
//
// The largest: values that may still be among them collect in the block's shared memory, as 64-bit keys (the value's
// bits in the order of values, then the index reversed: one comparison has both).  What may be is bounded from
// below: if r lanes of each of the 8 warps have met a value of at least b, then 8 r values are that large, and
// with 8 r >= `top` nothing below b is wanted -- r lanes by r maxima over a warp when one of its lanes has met a larger value,
// the smallest of the warps' bounds; warps read one another's without waiting, as bounds only grow.  Some tens of values are
// left at the end; each counts the larger ones, which is its place.  Where so many qualify that the memory
// would not hold them (rising rows, values all alike) the row is walked a second time, the block together.
//
// A row is a cluster's of 1 to 8 blocks (as many as the GPU has room for when rows are few); parts meet in the
// first block in a fixed order, so a row's results do not depend on the other rows' values nor on who came first.
// Bound by reading the logits, then by what a value costs beside its load: float32 rows of 65,536, 2,047 of them (537 MB,
// 82 us at a copy's bandwidth), take 90 us without alternatives, 98 with five, 114 with twenty (a bound of more lanes
// needs more maxima over a warp, and more values pass it).  64 rows with twenty take 13 us of 3, one row 4 without
// alternatives and 7 with twenty: a chain of the first loads, the warps' first bound, the cluster's meeting and the places.
#include "common.cuh"

#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_MAX_CLUSTER 8
#define LP_RESIDENT 4                  // blocks of a multiprocessor
#define LP_LOG2E 1.4426950408889634f
#define LP_LN2 0.6931471805599453f

#define LP_ROOM 640                    // values that a block can collect

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

struct __align__(16) LpPart { float m, s, w; int above; };

__device__ __forceinline__ float lp_ref(float m) { return m == -INFINITY ? 0.f : m; }
// From one reference to a larger one, in units of log2; far ones stay finite (2^-300 is 0).
__device__ __forceinline__ float lp_move(float from, float to) { return fmaxf((from - to) * LP_LOG2E, -300.f); }
// A warp's lanes put together, always in the same order: to the largest reference, then sums.
__device__ __forceinline__ LpPart lp_meet(const LpPart& a) {
    LpPart p;
    p.m = rv_warp_max(a.m);
    p.s = p.w = 0.f;
    if (a.s != 0.f) {
        const float d = lp_move(lp_ref(a.m), lp_ref(p.m)), f = lp_exp2(d);
        p.s = a.s * f;
        p.w = (a.w + a.s * d) * f;
    }
    p.s = rv_warp_sum(p.s);
    p.w = rv_warp_sum(p.w);
    p.above = __reduce_add_sync(0xffffffffu, a.above);
    return p;
}

template <bool TOP> struct LpShared {
    LpPart part[LP_WARPS];
    LpPart whole;
};
template <> struct LpShared<true> {
    LpPart part[LP_WARPS];
    LpPart whole;
    u64 room[LP_ROOM], left[LP_ROOM];
    u64 best[LP_MAX_CLUSTER][32];      // the parts' largest, descending; [0] is what this block leaves
    unsigned bound[LP_WARPS];
    int count, kept;
};

// Places `n` keys of `from` by how many are larger; the first `top` of them go to `to`, the rest of `to` is 0.
__device__ __forceinline__ void lp_place(const u64* from, int n, int top, u64* to) {
    __syncthreads();
    if (threadIdx.x >= n && threadIdx.x < 32) to[threadIdx.x] = 0ull;
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const u64 x = from[i];
        int larger = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) larger += from[j] > x;
        if (larger < 32) to[larger] = larger < top ? x : 0ull;
    }
    __syncthreads();
}

template <typename T, bool TOP>
struct LpThread {
    static constexpr int N = LpVec<T>::N, U = LpVec<T>::UNROLL, E = N * U;
    float m = -INFINITY, s = 0.f, w = 0.f, limit = -INFINITY;
    int above = 0;
    bool first = true;
    float given;
    int top;
    u64 least = 0ull;                  // only larger keys are wanted
    LpShared<TOP>& sh;

    __device__ __forceinline__ LpThread(LpShared<TOP>& shared, int k) : top(k), sh(shared) {}

    // Of E values: the sums; the largest.
    __device__ __forceinline__ float sums(const float (&x)[E]) {
        float bm = x[0];
#pragma unroll
        for (int i = 1; i < E; ++i) bm = fmaxf(bm, x[i]);
        if (bm > m) {
            if (s != 0.f) {
                const float d = lp_move(m, bm), f = lp_exp2(d);
                w = (w + s * d) * f;
                s *= f;
            }
            m = bm;
        }
        const float c = lp_ref(m);
        float s2[2] = {0.f, 0.f}, w2[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < E; ++i) {
            // (far below: 2^u is 0, and so is its product with u)
            const float u = lp_max_nan((x[i] - c) * LP_LOG2E, -200.f), e = lp_exp2(u);
            s2[i & 1] += e;
            w2[i & 1] = fmaf(e, u, w2[i & 1]);
            above += x[i] > given;
        }
        s += s2[0] + s2[1];
        w += w2[0] + w2[1];
        return bm;
    }
    // The r-th largest of a warp's lanes.
    __device__ __forceinline__ unsigned rth(unsigned mine, int r) const {
        unsigned b = 0u;
        for (int k = 0; k < r; ++k) {
            b = __reduce_max_sync(0xffffffffu, mine);
            const unsigned who = __ballot_sync(0xffffffffu, mine == b);
            if ((int)(threadIdx.x & 31) == __ffs(who) - 1) mine = 0u;
        }
        return b;
    }
    template <typename Col, typename Real>
    __device__ __forceinline__ void collect(const float (&x)[E], float limit, Col col, Real real) {
        // (few lanes have any, and one at most: a loop over them is shorter than their code written out, which costs more to fetch
        // than to run)
        unsigned which = 0u;
#pragma unroll
        for (int i = 0; i < E; ++i) which |= x[i] >= limit ? 1u << i : 0u;
        while (which) {
            const int i = __ffs(which) - 1;
            which &= which - 1;
            float v[E];
#pragma unroll
            for (int k = 0; k < E; ++k) v[k] = x[k];
#pragma unroll
            for (int h = E / 2; h > 0; h >>= 1)
#pragma unroll
                for (int k = 0; k < h; ++k) v[k] = (i & h) ? v[k + h] : v[k];
            const u64 key = ((u64)lp_key(v[0]) << 32) | (0xffffffffu - (unsigned)col(i));
            if (key > least && real(i)) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < LP_ROOM) sh.room[at] = key;
            }
        }
    }
    // Adds E values of this thread (the whole block comes here): x[i] is column col(i), if real(i).
    template <typename Col, typename Real>
    __device__ __forceinline__ void take(const float (&x)[E], Col col, Real real) {
        const float was = m, bm = sums(x);
        if constexpr (TOP) {
            const int lane = threadIdx.x & 31;
            // (below the limit nothing is wanted, nor does it change the warp's bound, which is not below the limit)
            if (first || __any_sync(0xffffffffu, bm >= limit)) {
                if (__any_sync(0xffffffffu, m > was)) {
                    const unsigned b = rth(m == -INFINITY ? 0u : lp_key(m), (top + LP_WARPS - 1) / LP_WARPS);
                    if (lane == 0) sh.bound[threadIdx.x >> 5] = b;
                    __syncwarp();
                }
                if (first) __syncthreads();                          // every warp has a bound
                first = false;
                // the warps' bounds as they are: they only grow, so older ones hold too
                const unsigned b = __reduce_min_sync(0xffffffffu, *(volatile unsigned*)&sh.bound[lane & (LP_WARPS - 1)]);
                limit = b ? lp_value(b) : -INFINITY;
                if (bm >= limit) collect(x, limit, col, real);
                __syncwarp();
            }
        }
    }
    // The same for the largest alone, a block together and never too many: what would overflow the memory is
    // taken again with the bound that the values in it give.
    template <typename Col, typename Real>
    __device__ __forceinline__ void take_again(const float (&x)[E], Col col, Real real) {
        const int before = sh.count;
        for (;;) {
            __syncthreads();
            collect(x, -INFINITY, col, real);
            __syncthreads();
            const int n = sh.count;
            if (n <= LP_ROOM / 2) break;
            lp_place(sh.room, min(n, LP_ROOM), top, sh.best[0]);
            least = sh.best[0][top - 1];
            if (n <= LP_ROOM) {                                      // all are here: keep the best
                if (threadIdx.x < top) sh.room[threadIdx.x] = sh.best[0][threadIdx.x];
            } else {
                --least;                                             // again, with the last of them let in
            }
            if (threadIdx.x == 0) sh.count = n <= LP_ROOM ? top : before;
            __syncthreads();
            if (n <= LP_ROOM) break;
        }
        __syncthreads();
    }
};

// Walks a row's part: `body(values, column of value i, whether there is one)` of every thread, round by round; the next round's
// values are requested before a round is taken.
// `ready()` comes behind the first requests.
template <typename T, typename Ready, typename Body>
__device__ __forceinline__ void lp_walk(const T* x, int vocab, int part, int parts, Ready ready, Body body) {
    constexpr int N = LpVec<T>::N, U = LpVec<T>::UNROLL, E = N * U, ROUND = U * LP_THREADS;
    const int tid = threadIdx.x;
    // whole 16-byte vectors from the first aligned one on, shared out over the parts; what lies
    // before and behind them is the last part's
    const int head = min(vocab, (int)((((16 - ((uintptr_t)x & 15)) & 15)) / sizeof(T)));
    const int vectors = (vocab - head) / N, tail = head + vectors * N;
    const int v0 = (int)((long long)vectors * part / parts), v1 = (int)((long long)vectors * (part + 1) / parts);
    const T* from = x + head;
    float next[E], v[E];
    auto load = [&](int at) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = at + u * LP_THREADS + tid;
            if (i < v1) {
                LpVec<T>::load(from + (size_t)i * N, next + u * N);
            } else {
#pragma unroll
                for (int k = 0; k < N; ++k) next[u * N + k] = -INFINITY;
            }
        }
    };
    if (v0 < v1) load(v0);
    ready();
    for (int at = v0; at < v1; at += ROUND) {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = next[i];
        if (at + ROUND < v1) load(at + ROUND);
        const int base = head + (at + tid) * N, mine = at + tid;
        body(v, [&](int i) { return base + (i / N) * LP_THREADS * N + i % N; },
             [&](int i) { return mine + (i / N) * LP_THREADS < v1; });
    }
    if (part == parts - 1 && head + vocab - tail > 0) {
        const int col = tid < head ? tid : tail + tid - head;
        const bool have = col < vocab;
        v[0] = have ? rv_load(x + col) : -INFINITY;
#pragma unroll
        for (int i = 1; i < E; ++i) v[i] = -INFINITY;
        body(v, [&](int) { return col; }, [&](int i) { return i == 0 && have; });
    }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS, LP_RESIDENT) token_logprobs_kernel(
    const T* __restrict__ logits, long long row_stride, int vocab, const int* __restrict__ tokens, int top,
    float* __restrict__ logprob, int* __restrict__ rank, float* __restrict__ entropy, float* __restrict__ top_logprob,
    int* __restrict__ top_id, int parts) {
    rv_pdl_prologue();
    __shared__ LpShared<TOP> sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long row = blockIdx.x / parts;
    const int part = (int)(blockIdx.x - row * parts);
    const T* x = logits + row * row_stride;
    if constexpr (TOP) {
        if (tid == 0) sh.count = sh.kept = 0;
        if (tid < LP_WARPS) sh.bound[tid] = 0u;
        __syncthreads();
    }
    const int token = tokens[row];
    const bool known = token >= 0 && token < vocab;
    LpThread<T, TOP> th(sh, top);
    lp_walk(x, vocab, part, parts, [&] { th.given = known ? rv_load(x + token) : INFINITY; },
            [&](auto& v, auto col, auto real) { th.take(v, col, real); });
    // ---- the warp's, the block's, the cluster's ------------------------------------------------
    {
        const LpPart p = lp_meet({th.m, th.s, th.w, th.above});
        if (lane == 0) sh.part[warp] = p;
    }
    __syncthreads();
    if (warp == LP_WARPS - 1) {
        const LpPart none = {-INFINITY, 0.f, 0.f, 0}, p = lp_meet(lane < LP_WARPS ? sh.part[lane] : none);
        if (lane == 0) sh.whole = p;
    }
    if constexpr (TOP) {
        const int n = sh.count;
        unsigned b = sh.bound[0];
#pragma unroll
        for (int k = 1; k < LP_WARPS; ++k) b = min(b, sh.bound[k]);
        if (n > LP_ROOM) {
            // rising values, or too many alike: the part once more
            __syncthreads();
            if (tid == 0) sh.count = 0;
            __syncthreads();
            th.least = b ? ((u64)b << 32) - 1ull : 0ull;
            lp_walk(x, vocab, part, parts, [] {}, [&](auto& v, auto col, auto real) { th.take_again(v, col, real); });
            lp_place(sh.room, sh.count, top, sh.best[0]);
        } else {
            // those that the last bound leaves
            for (int i = tid; i < n; i += LP_THREADS)
                if ((unsigned)(sh.room[i] >> 32) >= b) sh.left[atomicAdd(&sh.kept, 1)] = sh.room[i];
            __syncthreads();
            lp_place(sh.left, sh.kept, top, sh.best[0]);
        }
    } else {
        __syncthreads();
    }
    if (parts > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (part == 0) {
            auto remote = [](const void* p, int rank_) {
                unsigned a;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((unsigned)__cvta_generic_to_shared(p)), "r"(rank_));
                return a;
            };
            if constexpr (TOP) {                                     // warp k brings part k's list
                if (warp > 0 && warp < parts) {
                    u64 key;
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(remote(&sh.best[0][lane], warp)) : "memory");
                    sh.best[warp][lane] = key;
                }
            }
            if (warp == 0) {
                // lane k brings part k's sums
                LpPart q = {-INFINITY, 0.f, 0.f, 0};
                if (lane < parts)
                    asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(q.m), "=f"(q.s), "=f"(q.w), "=r"(q.above) : "r"(remote(&sh.whole, lane)) : "memory");
                q = lp_meet(q);
                __syncwarp();
                if (lane == 0) sh.whole = q;
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");     // nobody leaves while it is read
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (part != 0) return;
    }
    const LpPart p = sh.whole;
    const float c = lp_ref(p.m), logs = logf(p.s);
    if (tid == 0) {
        const float h = logs - LP_LN2 * (p.w / p.s);
        logprob[row] = known ? (th.given - c) - logs : NAN;
        rank[row] = known ? p.above + 1 : 0;
        entropy[row] = h < 0.f ? 0.f : h;
    }
    if constexpr (TOP) {
        // a key of part `warp`: its place is how many of all the parts' are larger
        const u64 key = warp < parts && lane < top ? sh.best[warp][lane] : 0ull;
        // (lists are in order: bisection in all of them at once)
        int place = lane;
        if (parts > 1) {
            int larger[LP_MAX_CLUSTER];
#pragma unroll
            for (int k = 0; k < LP_MAX_CLUSTER; ++k) larger[k] = 0;
            for (int step = top == 32 ? 16 : 1 << (31 - __clz(top)); step > 0; step >>= 1)
#pragma unroll
                for (int k = 0; k < LP_MAX_CLUSTER; ++k)
                    larger[k] += (sh.best[k][larger[k] + step - 1] > key) ? step : 0;
            place = 0;
#pragma unroll
            for (int k = 0; k < LP_MAX_CLUSTER; ++k) place += k < parts ? larger[k] + (sh.best[k][larger[k]] > key) : 0;   // (31 + 1)
        }
        if (key != 0ull && place < top) {
            top_logprob[row * top + place] = (lp_value((unsigned)(key >> 32)) - c) - logs;
            top_id[row * top + place] = (int)(0xffffffffu - (unsigned)key);
        }
        const int have = __syncthreads_count(key != 0ull);
        if (tid < top && tid >= have) {                               // places that nothing takes
            top_logprob[row * top + tid] = NAN;
            top_id[row * top + tid] = -1;
        }
    }
}

// Arguments packed, 8 bytes each, as the calls of cache_8bit.cu.
struct LpCall {
    const void* logits;
    const int* tokens;
    float* logprob;
    int* rank;
    float *entropy, *top_logprob;
    int* top_id;
    void* stream;
    long long dtype, row_stride, rows, vocab, top;
};
extern "C" int rv_token_logprobs(const LpCall* c) {
    const void* logits = c->logits;
    const int* tokens = c->tokens;
    float *logprob = c->logprob, *entropy = c->entropy, *top_logprob = c->top_logprob;
    int *rank = c->rank, *top_id = c->top_id;
    void* stream = c->stream;
    const long long row_stride = c->row_stride;
    const int dtype = (int)c->dtype, rows = (int)c->rows, vocab = (int)c->vocab, top = (int)c->top;
    if (c->rows > 0x7fffffff || c->vocab > 0x7fffffff) RV_FAIL("token_logprobs: bad sizes");
    if (rows == 0) return 0;
    if (rows < 0 || vocab <= 0) RV_FAIL("token_logprobs: bad sizes");
    if (top < 0 || top > 32 || top > vocab) RV_FAIL("token_logprobs: %d alternatives (0 to 32, at most the vocabulary)", top);
    // blocks a row: as many as the GPU holds at once, a round of loads each at least
    const int size = dtype == RV_DTYPE_F32 ? 4 : 2, sms = rv_sm_count();
    int parts = 1;
    while (2 * parts <= LP_MAX_CLUSTER && (long long)rows * 2 * parts <= (long long)LP_RESIDENT * sms &&
           (long long)vocab * size >= (long long)2 * parts * LP_THREADS * 64)
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
