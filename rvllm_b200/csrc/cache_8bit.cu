// Keys and values in 8 bits: the write of a step's rows into the paged cache, and pages read back.
//
// A page holds int8 [kv heads][page size][head size], and each (page, head) one float32 scale s, a power of two:
// the value that q stands for is q * s.  s = 2^e for the smallest e in [-60, 60] with max |x| <= 127 * 2^e over the
// block's finite values; q = rint(x / s), clamped to [-127, 127]; NaN becomes 0, an infinity +-127.  Powers of
// two: then q * s is a bfloat16 exactly (what the tensor cores are fed carries no second rounding), x / s is exact, and a
// block whose scale has to grow loses at most the bits that the larger scale drops.  A finer scale, max |x| / 127, would
// halve a block's rounding error at best (a quarter on average) and lose the three.
//
// A page is filled from its first slot on.  A call that writes slot 0 begins the page anew: its scale comes from
// the call's rows alone, whatever an earlier holder of the page left.  Otherwise the scale is the larger
// of the old one and what the rows need, and where it grew the other slots become rint(q * old / new).
// A page's tokens stand together in the call (nothing but tokens without a slot between them): the block of a run settles its page's
// scale alone, and two of them would both change one page.  Nothing looks for that: blocks that hold every run's page against
// all later ones took 3 of a short call's 4 us, 24 us at 2,048 tokens.
//
// One kernel.  A lane has 8 dimensions of a head's first half and the 8 that they turn with, so a warp has
// 32 / (head size / 16) heads at a time: of one token for the queries; for keys and values of as many tokens, one
// head.  A block of the latter takes a range of tokens, up to 32, and of it the pages that begin there, to their last
// token in the call.  The rows are read once (two rounds of them stay in shared memory, a thread its own: the largest of a page
// has to be known before any is written), the pages' scales settled a lane each, then the rows written.
//
// What bounds it: what a block does beside its rows (whose tokens and pages they are, the pages' largest values, two
// meetings of its warps) and four reads that wait for one another (slots, positions, angles and rows, scales), for as many
// waves of blocks as there are; registers leave a multiprocessor four or five.  32 / 8 heads of 64: 64 tokens 4.2 us,
// 2,048 tokens 11.4 us, 8,192 tokens 44 us; their bytes at a copy's bandwidth 0.1, 3.5 and 14 us.
#include <cuda_fp16.h>

#include "common.cuh"

#define C8_MAX_HEAD 256
#define C8_WARPS 4

struct C8Write {
    const void* rows;                  // [tokens][heads q | kv heads k | kv heads v], `row_stride` elements apart
    void* q_out;                       // [tokens][heads * head size]
    const float *q_weight, *k_weight, *cos_table, *sin_table;
    const int *positions, *slots;
    signed char *k_cache, *v_cache;
    float *k_scale, *v_scale;
    long long row_stride, total_slots, table_rows;
    float eps;
    int n_tokens, num_heads, num_kv_heads, head_dim, page_size, page_shift, aligned, range;
    long long kv_blocks;
};

__device__ __forceinline__ void c8_load8(const float* p, bool vec, float (&v)[8]) {
    if (vec) {
        const float4 a = *(const float4*)p, b = *(const float4*)(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p[i];
    }
}
__device__ __forceinline__ void c8_load8(const __nv_bfloat16* p, bool vec, float (&v)[8]) {
    if (vec) {
        const uint4 raw = *(const uint4*)p;
        const __nv_bfloat162* h = (const __nv_bfloat162*)&raw;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __bfloat1622float2(h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
    }
}
__device__ __forceinline__ void c8_store8(float* p, bool vec, const float (&v)[8]) {
    if (vec) {
        *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*)(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = v[i];
    }
}
__device__ __forceinline__ void c8_store8(__nv_bfloat16* p, bool vec, const float (&v)[8]) {
    if (vec) {
        uint4 raw;
        __nv_bfloat162* h = (__nv_bfloat162*)&raw;
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *(uint4*)p = raw;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(v[i]);
    }
}

// The smallest e in [-60, 60] with most <= 127 * 2^e (127 = 1.984375 * 2^6), most >= 0 and finite.
__device__ __forceinline__ int c8_exponent(float most) {
    const unsigned b = __float_as_uint(most);
    const int e = (int)((b + (0x7fffffu - 0x7e0000u)) >> 23) - 127 - 6;
    return max(-60, min(60, e));
}
__device__ __forceinline__ float c8_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// Sum over the `lph` lanes from `lane0` on that have a head.
template <typename A>
__device__ __forceinline__ A c8_sum(A v, int lane0, int lph) {
    if ((lph & (lph - 1)) == 0) {
        for (int o = lph >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    A sum = 0;
    for (int k = 0; k < lph; ++k) sum += __shfl_sync(0xffffffffu, v, (lane0 + k) & 31);
    return sum;
}

// To float32, to odd: cut off, the last bit set where something was.  What is rounded to eight bits and what is held against 127 steps
// afterwards comes out as if float64 had been.
__device__ __forceinline__ float c8_odd(double v) {
    // (29 bits go; below 2^-126 more do, of what is zero in eight bits)
    return __uint_as_float(__float_as_uint(__double2float_rz(v)) | ((__double2loint(v) & 0x1fffffff) != 0));
}
// One key or value head of one token: norm and rotation in float64, so that what a page holds is the formula's value, whatever
// the order of the sums (float32 throughout left ten values in a million on the wrong side of a border between two steps,
// rounding to the nearest float32 first one).
template <typename T>
__device__ __forceinline__ void c8_head(const C8Write& a, const T* src, const float* w, bool turn, int t, bool live, int d0,
                                        int lane0, int lph, float (&x)[8], float (&y)[8]) {
    const int half = a.head_dim >> 1;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = y[i] = 0.f;
    if (live) {
        c8_load8(src + d0, a.aligned, x);
        c8_load8(src + half + d0, a.aligned, y);
    }
    if (!w && !turn) return;
    double inv = 1.0;
    if (w) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += (double)x[i] * x[i] + (double)y[i] * y[i];
        inv = 1.0 / sqrt(c8_sum(ss, lane0, lph) / a.head_dim + (double)a.eps);
    }
    if (!live) return;
    float wx[8], wy[8], c[8], s[8];
    if (w) {
        c8_load8(w + d0, a.aligned, wx);
        c8_load8(w + half + d0, a.aligned, wy);
    }
    bool angle = turn;
    if (turn) {
        const long long p = a.positions[t];
        angle = p >= 0 && p < a.table_rows;
        if (angle) {
            c8_load8(a.cos_table + p * half + d0, a.aligned, c);
            c8_load8(a.sin_table + p * half + d0, a.aligned, s);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        double u = x[i], v = y[i];
        if (w) {
            u = u * inv * wx[i];
            v = v * inv * wy[i];
        }
        if (angle) {
            const double turned = u * c[i] - v * s[i];
            v = u * s[i] + v * c[i];
            u = turned;
        }
        x[i] = turn && !angle ? NAN : c8_odd(u);                  // (held as 0)
        y[i] = turn && !angle ? NAN : c8_odd(v);
    }
}

// Query heads h0, h0 + per, ... of token t: the token's angles and the weights are read once, all rows requested before any is
// used.
template <typename T, int ROUNDS>
__device__ __forceinline__ void c8_queries(const C8Write& a, int t, int h0, int per, bool mine, int d0, int lane0, int lph) {
    const int half = a.head_dim >> 1;
    const T* src = (const T*)a.rows + (size_t)t * a.row_stride;
    T* dst = (T*)a.q_out + (size_t)t * a.num_heads * a.head_dim;
    float x[ROUNDS][8], y[ROUNDS][8], wx[8], wy[8], c[8], s[8];
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const int h = h0 + k * per;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[k][i] = y[k][i] = 0.f;
        if (mine && h < a.num_heads) {
            c8_load8(src + (size_t)h * a.head_dim + d0, a.aligned, x[k]);
            c8_load8(src + (size_t)h * a.head_dim + half + d0, a.aligned, y[k]);
        }
    }
    if (a.q_weight) {
        c8_load8(a.q_weight + d0, a.aligned, wx);
        c8_load8(a.q_weight + half + d0, a.aligned, wy);
    }
    const bool turn = a.cos_table != nullptr;
    bool angle = false;
    if (turn) {
        const long long p = a.positions[t];
        angle = p >= 0 && p < a.table_rows;
        if (angle) {
            c8_load8(a.cos_table + p * half + d0, a.aligned, c);
            c8_load8(a.sin_table + p * half + d0, a.aligned, s);
        }
    }
#pragma unroll
    for (int k = 0; k < ROUNDS; ++k) {
        const int h = h0 + k * per;
        if (a.q_weight) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss += x[k][i] * x[k][i] + y[k][i] * y[k][i];
            const float inv = 1.f / sqrtf(c8_sum(ss, lane0, lph) / (float)a.head_dim + a.eps);       // one division for sixteen
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                x[k][i] = x[k][i] * inv * wx[i];
                y[k][i] = y[k][i] * inv * wy[i];
            }
        }
        if (turn)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = x[k][i], v = y[k][i];
                x[k][i] = angle ? u * c[i] - v * s[i] : NAN;       // (a position outside the table has no angle)
                y[k][i] = angle ? u * s[i] + v * c[i] : NAN;
            }
        if (mine && h < a.num_heads) {
            c8_store8(dst + (size_t)h * a.head_dim + d0, a.aligned, x[k]);
            c8_store8(dst + (size_t)h * a.head_dim + half + d0, a.aligned, y[k]);
        }
    }
}

// The largest |x|, `most` among them; NaN if any is.
__device__ __forceinline__ float c8_most(const float (&x)[8], float most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(most) : "f"(fabsf(x[i])));
    return most;
}
__device__ __forceinline__ float c8_most_finite(const float (&x)[8], float most) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float v = fabsf(x[i]);
        if (v <= 3.402823466e38f) most = fmaxf(most, v);
    }
    return most;
}
// rint(x / scale).  `plain`: all are within 127 scales, and the sum with 1.5 * 2^23 has the whole number in its last byte
// (x * inv is exact, so that this rounds once, half to even).
__device__ __forceinline__ uint2 c8_pack(const float (&x)[8], float inv, bool plain) {
    unsigned u[2] = {0u, 0u};
    if (plain) {
        unsigned b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(fmaf(x[i], inv, 12582912.f));
#pragma unroll
        for (int i = 0; i < 2; ++i)
            u[i] = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040), 0x5410);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int q = max(-127, min(127, __float2int_rn(x[i] * inv)));     // NaN: 0
            u[i >> 2] |= (unsigned)(q & 0xff) << (8 * (i & 3));
        }
    }
    return make_uint2(u[0], u[1]);
}

// What a block knows of the pages that begin in its range.
struct C8Runs {
    unsigned most[32];                 // bits of the largest finite |x| of each
    float inv[32];                     // 1 / scale
    int lowest[32];                    // first slot written
    int page[32];
    unsigned slots[32][2];             // those written, modulo 64
    int twice;                         // one of them twice, it may be
};

// `MANY`: for as many tokens as fill the GPU several times over.  Then blocks of a multiprocessor count (five: 96 registers a
// thread), and a warp has two rounds of a token's query heads; else what a thread can request at once (us so / the other way:
// 32 / 8 heads of 64, 64 tokens 4.1 / 4.4, 512 5.1 / 5.2, 2,048 12.5 / 11.4, 8,192 48.0 / 43.6).
template <typename T, bool MANY>
__global__ void __launch_bounds__(C8_WARPS * 32, MANY ? 5 : 4) qk_norm_rope_write_8bit_kernel(const __grid_constant__ C8Write a) {
    rv_pdl_prologue();
    __shared__ C8Runs run;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int lph = a.head_dim >> 4, per = 32 / lph;           // lanes a head, heads a warp
    const int sub = lane / lph, d0 = (lane - sub * lph) * 8, lane0 = sub * lph;
    const int half = a.head_dim >> 1;
    __align__(16) float x[8], y[8];
    if ((long long)blockIdx.x >= a.kv_blocks) {
        // ---- query heads --------------------------------------------------------------------
        const long long id = ((long long)blockIdx.x - a.kv_blocks) * C8_WARPS + warp;
        constexpr int ROUNDS = MANY ? 2 : 1;
        const int shares = (a.num_heads + per * ROUNDS - 1) / (per * ROUNDS);
        const long long t = id / shares;
        if (t >= a.n_tokens) return;
        c8_queries<T, ROUNDS>(a, (int)t, (int)(id - t * shares) * per * ROUNDS + sub, per, sub < per, d0, lane0, lph);
        return;
    }
    // ---- one key or value head of the pages that begin within a range of tokens ---------------
    const int pairs = 2 * a.num_kv_heads;
    const int first = (int)((long long)blockIdx.x / pairs) * a.range, pair = (int)((long long)blockIdx.x % pairs);
    const bool is_k = pair < a.num_kv_heads;
    const int g = is_k ? pair : pair - a.num_kv_heads;
    const T* src = (const T*)a.rows + (size_t)(a.num_heads + pair) * a.head_dim;
    const float* w = is_k ? a.k_weight : nullptr;
    const bool turn = is_k && a.cos_table != nullptr;
    signed char* cache = is_k ? a.k_cache : a.v_cache;
    float* scales = is_k ? a.k_scale : a.v_scale;
    auto slot_of = [&](int t) {
        const int s = t >= 0 && t < a.n_tokens ? a.slots[t] : -1;
        return s >= 0 && s < a.total_slots ? s : -1;
    };
    auto page_of = [&](int s) { return a.page_shift >= 0 ? s >> a.page_shift : s / a.page_size; };
    // (every warp finds the same pages)
    const unsigned full = 0xffffffffu, below = (1u << lane) - 1u;
    // this window's tokens, and the page of the last token with a slot before it
    const int mine = slot_of(first + lane);
    int back = slot_of(first - 1 - lane);
    const int my_page = mine >= 0 ? page_of(mine) : -1;
    const unsigned real = __ballot_sync(full, mine >= 0);
    int before = -1;
    for (int at = first - 1;;) {
        const unsigned have = __ballot_sync(full, back >= 0);
        if (have) {
            before = page_of(__shfl_sync(full, back, __ffs(have) - 1));
            break;
        }
        at -= 32;
        if (at < 0) break;
        back = slot_of(at - lane);
    }
    const unsigned earlier = real & below;
    int prev = __shfl_sync(full, my_page, earlier ? 31 - __clz(earlier) : 0);
    if (!earlier) prev = before;
    const bool changes = mine >= 0 && my_page != prev;
    const unsigned begins = __ballot_sync(full, changes);
    const unsigned owned = begins & (a.range < 32 ? (1u << a.range) - 1u : full);
    if (!owned) return;                                        // (the whole block)
    const int n_runs = __popc(owned), l0 = __ffs(owned) - 1, last = 31 - __clz(owned);
    // tokens [t0, t1): up to the first token behind the range that has a slot of another page
    const int t0 = first + l0;
    int t1 = first + 32;
    {
        const unsigned after = begins & ~((2u << last) - 1u);
        const int last_page = __shfl_sync(full, my_page, last);
        if (after) {
            t1 = first + __ffs(after) - 1;
        } else {
            for (bool more = t1 < a.n_tokens; more;) {
                const int s = slot_of(t1 + lane);
                const unsigned stop = __ballot_sync(full, (s >= 0 && page_of(s) != last_page) || t1 + lane >= a.n_tokens);
                t1 += stop ? __ffs(stop) - 1 : 32;
                more = !stop;
            }
            t1 = min(t1, a.n_tokens);
        }
    }
    if (warp == 0) {
        run.most[lane] = 0u;
        run.lowest[lane] = a.page_size;
        run.slots[lane][0] = run.slots[lane][1] = 0u;
        run.twice = 0;
        if ((owned >> lane) & 1u) run.page[__popc(owned & below)] = my_page;
    }
    __syncthreads();
    // lane i looks after run i: its page and what its scale was
    const int page_i = lane < n_runs ? run.page[lane] : 0;
    const size_t block_i = (size_t)page_i * a.num_kv_heads + g;
    const float old = lane < n_runs ? scales[block_i] : 0.f;
    // A group of lanes a token: `slot` (-1: none) and the number of its run.
    auto whose = [&](int t, int& slot, int& number) {
        const int in = t - first;
        const int s = __shfl_sync(full, mine, in & 31);
        slot = in < 32 ? s : slot_of(t);
        if (sub >= per || t >= t1) slot = -1;
        number = in < 32 ? __popc(owned & ((2u << in) - 1u)) - 1 : n_runs - 1;
    };
    constexpr int HOLD = 2;             // rounds whose rows are kept: a range and the page that it ends in
    const int step = C8_WARPS * per, begin = t0 + warp * per;
    __shared__ float4 held_rows[HOLD * 4][C8_WARPS * 32];
    float hm[HOLD], m;                  // the largest |x| of each, or NaN
    auto measure = [&](int t, int slot, int number, float (&u)[8], float (&v)[8], float& whole) {
        c8_head(a, src + (size_t)(slot >= 0 ? t : t0) * a.row_stride, w, turn, t, slot >= 0, d0, lane0, lph, u, v);
        float most = whole = c8_most(v, c8_most(u, 0.f));
        if (!(most <= 3.402823466e38f)) most = c8_most_finite(v, c8_most_finite(u, 0.f));
        if (slot >= 0) {
            atomicMax(&run.most[number], __float_as_uint(most));
            if (d0 == 0) {
                const unsigned in = slot - page_of(slot) * a.page_size, bit = 1u << (in & 31u);
                atomicMin(&run.lowest[number], (int)in);
                if (atomicOr(&run.slots[number][(in >> 5) & 1u], bit) & bit) run.twice = 1;
            }
        }
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
        if (begin + i * step < t1) {
            int slot, number;
            whose(begin + i * step + sub, slot, number);
            measure(begin + i * step + sub, slot, number, x, y, hm[i]);
            held_rows[4 * i][threadIdx.x] = *(const float4*)x;
            held_rows[4 * i + 1][threadIdx.x] = *(const float4*)(x + 4);
            held_rows[4 * i + 2][threadIdx.x] = *(const float4*)y;
            held_rows[4 * i + 3][threadIdx.x] = *(const float4*)(y + 4);
        }
    for (int t = begin + HOLD * step; t < t1; t += step) {
        int slot, number;
        whose(t + sub, slot, number);
        measure(t + sub, slot, number, x, y, m);
    }
    __syncthreads();
    bool grows = false;
    float ratio = 0.f;
    if (lane < n_runs) {
        float s = c8_pow2(c8_exponent(__uint_as_float(run.most[lane])));
        if (run.lowest[lane] > 0) {
            s = fmaxf(old, s);
            grows = s != old;
            ratio = old / s;
        }
        if (warp == 0) {
            scales[block_i] = s;
            run.inv[lane] = 1.f / s;
        }
    }
    // pages whose scale grew: what they hold follows (the slots written below too, which does no harm)
    for (unsigned todo = __ballot_sync(full, grows); todo; todo &= todo - 1) {
        const int i = __ffs(todo) - 1;
        const float by = __shfl_sync(full, ratio, i);
        signed char* held = cache + ((size_t)__shfl_sync(full, page_i, i) * a.num_kv_heads + g) * a.page_size * a.head_dim;
        for (int at = threadIdx.x * 16; at < a.page_size * a.head_dim; at += C8_WARPS * 512) {
            int4 v = *(const int4*)(held + at);
            signed char* b = (signed char*)&v;
#pragma unroll
            for (int k = 0; k < 16; ++k) b[k] = (signed char)__float2int_rn((float)b[k] * by);
            *(int4*)(held + at) = v;
        }
    }
    __syncthreads();
    auto store = [&](int t, int slot, int number, const float (&u)[8], const float (&v)[8], float whole) {
        // (of two tokens with one slot the later one is written)
        const int page = page_of(slot);
        bool later = false;
        if (slot >= 0 && run.twice)
            for (int k = t + 1; k < t1 && !later; ++k) {
                const int s = slot_of(k);
                if (s >= 0 && page_of(s) != page) break;
                later = s == slot;
            }
        if (slot >= 0 && !later) {
            const float inv = run.inv[number];
            const bool plain = whole * inv <= 127.f;
            signed char* dst = cache + (((size_t)page * a.num_kv_heads + g) * a.page_size + (slot - page * a.page_size)) * a.head_dim;
            *(uint2*)(dst + d0) = c8_pack(u, inv, plain);
            *(uint2*)(dst + half + d0) = c8_pack(v, inv, plain);
        }
    };
#pragma unroll
    for (int i = 0; i < HOLD; ++i)
        if (begin + i * step < t1) {
            int slot, number;
            whose(begin + i * step + sub, slot, number);
            *(float4*)x = held_rows[4 * i][threadIdx.x];
            *(float4*)(x + 4) = held_rows[4 * i + 1][threadIdx.x];
            *(float4*)y = held_rows[4 * i + 2][threadIdx.x];
            *(float4*)(y + 4) = held_rows[4 * i + 3][threadIdx.x];
            store(begin + i * step + sub, slot, number, x, y, hm[i]);
        }
    for (int t = begin + HOLD * step; t < t1; t += step) {
        int slot, number;
        whose(t + sub, slot, number);
        c8_head(a, src + (size_t)(slot >= 0 ? t + sub : t0) * a.row_stride, w, turn, t + sub, slot >= 0, d0, lane0, lph, x, y);
        store(t + sub, slot, number, x, y, c8_most(y, c8_most(x, 0.f)));
    }
}

// The entry points take their arguments packed, 8 bytes each (addresses, then sizes, then numbers), in the order of these
// records: a host call that hands over twenty arguments one by one takes 2 us, a record 0.4.
struct C8WriteCall {
    const void* rows;
    const float *q_weight, *k_weight, *cos_table, *sin_table;
    const int *positions, *slots;
    void *q_out, *k_cache, *v_cache;
    float *k_scale, *v_scale;
    void* stream;
    long long dtype, row_stride, n_tokens, num_heads, num_kv_heads, head_dim, table_rows, pages, page_size;
    double eps;
};
extern "C" int rv_qk_norm_rope_write_8bit(const C8WriteCall* c) {
    const void* rows = c->rows;
    const float *q_weight = c->q_weight, *k_weight = c->k_weight, *cos_table = c->cos_table, *sin_table = c->sin_table;
    const int *positions = c->positions, *slots = c->slots;
    void *q_out = c->q_out, *k_cache = c->k_cache, *v_cache = c->v_cache, *stream = c->stream;
    float *k_scale = c->k_scale, *v_scale = c->v_scale, eps = (float)c->eps;
    const long long row_stride = c->row_stride, table_rows = c->table_rows, pages = c->pages;
    const int dtype = (int)c->dtype, num_heads = (int)c->num_heads, num_kv_heads = (int)c->num_kv_heads;
    const int head_dim = (int)c->head_dim, page_size = (int)c->page_size, n_tokens = (int)c->n_tokens;
    if (c->n_tokens > 0x7fffffff || c->num_heads > 65535 || c->num_kv_heads > 65535 || c->page_size > 0x7fffffff)
        RV_FAIL("qk_norm_rope_write_8bit: bad sizes");
    if (n_tokens == 0) return 0;
    if (n_tokens < 0 || num_heads <= 0 || num_kv_heads <= 0 || page_size <= 0 || pages < 0)
        RV_FAIL("qk_norm_rope_write_8bit: bad sizes");
    if (head_dim <= 0 || head_dim % 16 || head_dim > C8_MAX_HEAD)
        RV_FAIL("qk_norm_rope_write_8bit: head size %d is not supported (a multiple of 16, at most %d)", head_dim, C8_MAX_HEAD);
    if (pages * page_size > 0x7fffffffLL) RV_FAIL("qk_norm_rope_write_8bit: more slots than int32 counts");
    if ((cos_table == nullptr) != (sin_table == nullptr) || (cos_table && !positions))
        RV_FAIL("qk_norm_rope_write_8bit: incomplete rotation table arguments");
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) % 16) RV_FAIL("qk_norm_rope_write_8bit: pages must be 16-byte aligned");
    C8Write a = {rows, q_out, q_weight, k_weight, cos_table, sin_table, positions, slots, (signed char*)k_cache,
                 (signed char*)v_cache, k_scale, v_scale, row_stride, pages * page_size, table_rows, eps, n_tokens,
                 num_heads, num_kv_heads, head_dim, page_size, (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1, 0, 0, 0};
    const int size = dtype == RV_DTYPE_F32 ? 4 : 2, per = 32 / (head_dim >> 4);
    a.aligned = ((uintptr_t)rows | (uintptr_t)q_out | (uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)cos_table |
                 (uintptr_t)sin_table) % 16 == 0 && row_stride * size % 16 == 0;
    a.range = C8_WARPS * per < 32 ? C8_WARPS * per : 32;
    a.kv_blocks = (long long)((n_tokens + a.range - 1) / a.range) * 2 * num_kv_heads;
    const bool many = n_tokens >= 8 * rv_sm_count();
    const int share = per * (many ? 2 : 1);                // of a token's query heads, a warp's
    const long long q_warps = (long long)n_tokens * ((num_heads + share - 1) / share);
    const long long blocks = a.kv_blocks + (q_warps + C8_WARPS - 1) / C8_WARPS;
    if (blocks > 0x7fffffffLL) RV_FAIL("qk_norm_rope_write_8bit: too many rows");
    RV_DISPATCH_DTYPE(dtype, "qk_norm_rope_write_8bit",
                      (rv_launch(many ? qk_norm_rope_write_8bit_kernel<T, true> : qk_norm_rope_write_8bit_kernel<T, false>, dim3((int)blocks), dim3(C8_WARPS * 32), 0,
                                 (cudaStream_t)stream, a)));
    RV_CHECK_LAUNCH("qk_norm_rope_write_8bit");
    return 0;
}

// ---- pages read back ----------------------------------------------------------------------------
// Page `ids[i]` as values.  A thread has 16 of them.  An id that is no page gives zeros.
template <typename T>
__global__ void __launch_bounds__(256) read_8bit_kernel(const signed char* __restrict__ cache, const float* __restrict__ scales,
                                                        const int* __restrict__ ids, T* __restrict__ out, long long total,
                                                        int heads, int head_bytes, long long pages) {
    rv_pdl_prologue();
    const long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 16;
    if (i >= total) return;
    const long long block = i / head_bytes, n = block / heads;
    const int page = ids[n];
    T* dst = out + i;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.f;
    if (page >= 0 && page < pages) {
        const long long from = (long long)page * heads + (block - n * heads);
        const float s = scales[from];
        const int4 raw = *(const int4*)(cache + from * head_bytes + (i - block * head_bytes));
        const signed char* b = (const signed char*)&raw;
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = (float)b[k] * s;
    }
#pragma unroll
    for (int k = 0; k < 16; k += 8) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = v[k + j];
        c8_store8(dst + k, true, w);
    }
}

struct C8ReadCall {
    const void* cache;
    const float* scales;
    const int* ids;
    void *out, *stream;
    long long dtype, n, heads, page_size, head_dim, pages;
};
extern "C" int rv_read_8bit(const C8ReadCall* c) {
    const void* cache = c->cache;
    void *out = c->out, *stream = c->stream;
    const float* scales = c->scales;
    const int* ids = c->ids;
    const long long pages = c->pages;
    const int dtype = (int)c->dtype, n = (int)c->n, heads = (int)c->heads, page_size = (int)c->page_size, head_dim = (int)c->head_dim;
    if (c->n > 0x7fffffff || c->heads > 65535 || c->page_size > 0x7fffffff) RV_FAIL("read_8bit: bad sizes");
    if (n == 0) return 0;
    if (n < 0 || heads <= 0 || page_size <= 0 || head_dim <= 0 || head_dim % 16) RV_FAIL("read_8bit: bad sizes");
    if (((uintptr_t)cache | (uintptr_t)out) % 16) RV_FAIL("read_8bit: pages must be 16-byte aligned");
    const long long head_bytes = (long long)page_size * head_dim, total = (long long)n * heads * head_bytes;
    const long long blocks = (total / 16 + 255) / 256;
    if (blocks > 0x7fffffffLL || head_bytes > 0x7fffffffLL) RV_FAIL("read_8bit: too many pages");
    RV_DISPATCH_DTYPE(dtype, "read_8bit",
                      (rv_launch(read_8bit_kernel<T>, dim3((int)blocks), dim3(256), 0, (cudaStream_t)stream,
                                 (const signed char*)cache, scales, ids, (T*)out, total, heads, (int)head_bytes, pages)));
    RV_CHECK_LAUNCH("read_8bit");
    return 0;
}

// ---- contexts widened for long portions ------------------------------------------------------------
// The keys and values that requests' portions may see, as pages of 64 tokens [page][64][kv heads][head size] and a block
// table for them, as the tcgen05 attention reads them: keys in bfloat16, values in float16 times a power of two of their page's
// own (attention_tcgen05.cu, RV_SCALED, says which).  Its blocks of 128 rows each read a request's whole context, so that
// one pass here costs less than widening the tiles in each of them (a prompt of 2,048 tokens, 32 / 8 heads of 64: 64
// blocks a head; 68 us with the tiles widened in place by three warps a block, which they keep waiting).  Exact,
// as scales are powers of two.
// `tile_exps`: the powers of the pages of 64, by request and place, marked in bit 16 where the exponents of the 8-bit pages within lie more
// than 32 apart; then `key_exps` has each key's.
// blockIdx.x: a page of 64, y: request, z: key/value head.  Slots behind the context are zeros, keys without a page NaN.
// Rows of a portion before position 0 are not the attention's: they are set to zero here.
struct C8Widen {
    const signed char *k, *v;
    const float *k_scale, *v_scale;
    const int *block_table, *q_start, *ctx_lens;
    __nv_bfloat16* wide_k;
    __half* wide_v;
    __nv_bfloat16* out;
    int *wide_table, *tile_exps;
    signed char* key_exps;
    long long pages;
    int max_blocks, first_req, num_heads, num_kv_heads, head_dim, page_size, window, width, room;
};
__global__ void __launch_bounds__(256) widen_8bit_kernel(const __grid_constant__ C8Widen a) {
    rv_pdl_prologue();
    const int i = blockIdx.y, r = a.first_req + i, g = blockIdx.z;
    const int clen = a.ctx_lens[r], qs = a.q_start[r], qlen = a.q_start[r + 1] - qs;
    const int lo = a.window > 0 ? max(0, clen - qlen - a.window + 1) : 0, b0 = lo / 64, b = b0 + blockIdx.x;
    if (blockIdx.x == 0)
        for (int k = threadIdx.x; k < a.width; k += 256) {
            const bool here = k >= b0 && k < b0 + a.room && (long long)k * 64 < clen && qlen > 0;
            if (g == 0) a.wide_table[(size_t)i * a.width + k] = here ? i * a.room + k - b0 : -1;
            if (!here) a.tile_exps[((size_t)i * a.width + k) * a.num_kv_heads + g] = 0;
        }
    if (blockIdx.x == 0 && clen < qlen) {
        const int per = a.num_heads / a.num_kv_heads * a.head_dim, pairs = per / 2;
        for (long long k = threadIdx.x; k < (long long)(qlen - clen) * pairs; k += 256) {
            const long long tok = k / pairs;
            ((unsigned*)(a.out + ((size_t)(qs + tok) * a.num_kv_heads + g) * per))[k - tok * pairs] = 0u;
        }
    }
    if ((long long)b * 64 >= clen || qlen <= 0) return;
    __shared__ int key_page[64], key_exp[64], most[2], least[2];
    if (threadIdx.x < 64) {
        const int key = b * 64 + threadIdx.x, blk = key / a.page_size;
        int page = key < clen && blk < a.max_blocks ? a.block_table[(size_t)r * a.max_blocks + blk] : -1;
        if (page >= a.pages) page = -1;
        const int e = page < 0 ? 0 : max(-60, min(60, (int)((__float_as_uint(a.v_scale[(size_t)page * a.num_kv_heads + g]) >> 23) & 0xff) - 127));
        key_page[threadIdx.x] = page;
        key_exp[threadIdx.x] = e;
        const int hi = __reduce_max_sync(0xffffffffu, page < 0 ? -999 : e), lo = __reduce_min_sync(0xffffffffu, page < 0 ? 999 : e);
        if ((threadIdx.x & 31) == 0) {
            most[threadIdx.x >> 5] = hi;
            least[threadIdx.x >> 5] = lo;
        }
    }
    __syncthreads();
    const int high = max(most[0], most[1]), spread = high - min(least[0], least[1]);
    const bool apart = spread > 32;
    const int tile_e = high == -999 ? 0 : high;
    if (threadIdx.x == 0 && b < a.width)
        a.tile_exps[((size_t)i * a.width + b) * a.num_kv_heads + g] = apart ? 0x10000 | (-8 & 0xffff) : (tile_e - 8) & 0xffff;
    if (apart && threadIdx.x < 64)
        a.key_exps[(((size_t)i * a.room + blockIdx.x) * a.num_kv_heads + g) * 64 + threadIdx.x] = (signed char)key_exp[threadIdx.x];
    const int pieces = a.head_dim / 16;
    for (int k = threadIdx.x; k < 64 * pieces; k += 256) {
        const int in = k / pieces, c = k - in * pieces, key = b * 64 + in, page = key_page[in];
        const bool ok = page >= 0;
        const size_t block = ok ? (size_t)page * a.num_kv_heads + g : 0;
        const size_t from = (block * a.page_size + (ok ? key % a.page_size : 0)) * a.head_dim + 16 * c;
        const size_t to = (((size_t)i * a.room + blockIdx.x) * 64 + in) * a.num_kv_heads * a.head_dim + (size_t)g * a.head_dim + 16 * c;
        const int4 zero = make_int4(0, 0, 0, 0);
        const int4 kr = ok ? *(const int4*)(a.k + from) : zero, vr = ok ? *(const int4*)(a.v + from) : zero;
        const float sk = ok ? a.k_scale[block] : key < clen ? NAN : 0.f, sv = c8_pow2(apart ? 8 : key_exp[in] - tile_e + 8);
        const signed char *kb = (const signed char*)&kr, *vb = (const signed char*)&vr;
#pragma unroll
        for (int h = 0; h < 16; h += 8) {
            float x[8];
            __align__(16) __half2 y[4];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (float)kb[h + j] * sk;
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = __floats2half2_rn((float)vb[h + 2 * j] * sv, (float)vb[h + 2 * j + 1] * sv);
            c8_store8(a.wide_k + to + h, true, x);
            *(uint4*)(a.wide_v + to + h) = *(const uint4*)y;
        }
    }
}

// Requests [first_req, first_req + n_reqs): `room` pages of 64 for each in `wide_k`, `wide_v` and `key_exps` [page][kv heads][64], `width`
// entries in `wide_table` and, a kv head each, in `tile_exps`.
extern "C" int rv_widen_8bit(const void* k_cache, const void* v_cache, const float* k_scale, const float* v_scale, long long pages,
                             const int* block_table, int max_blocks, const int* q_start, const int* ctx_lens, void* wide_k,
                             void* wide_v, int* wide_table, int* tile_exps, signed char* key_exps, int width, int room, void* out,
                             int first_req, int n_reqs, int num_heads,
                             int num_kv_heads, int head_dim, int page_size, int window, void* stream) {
    if (n_reqs == 0) return 0;
    if (n_reqs < 0 || n_reqs > 65535 || num_heads <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535 || num_heads % num_kv_heads ||
        head_dim <= 0 || head_dim % 16 || page_size <= 0 || window < 0 || width < 0 || room <= 0)
        RV_FAIL("widen_8bit: bad sizes");
    if (((uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)wide_k | (uintptr_t)wide_v) % 16)
        RV_FAIL("widen_8bit: pages must be 16-byte aligned");
    const C8Widen a = {(const signed char*)k_cache, (const signed char*)v_cache, k_scale, v_scale, block_table, q_start, ctx_lens,
                       (__nv_bfloat16*)wide_k, (__half*)wide_v, (__nv_bfloat16*)out, wide_table, tile_exps, key_exps, pages, max_blocks, first_req,
                       num_heads, num_kv_heads, head_dim, page_size, window, width, room};
    rv_launch(widen_8bit_kernel, dim3(room, n_reqs, num_kv_heads), dim3(256), 0, (cudaStream_t)stream, a);
    RV_CHECK_LAUNCH("widen_8bit");
    return 0;
}
