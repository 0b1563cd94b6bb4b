// Paged causal attention over keys and values held in 8 bits (cache_8bit.cu: int8 [pages][kv heads][page size]
// [head size], one power-of-two scale per page and head), single tokens and portions of prompts.  Compiled for one head
// size at a time (RV_HD: a multiple of 16, at most 256).
//
// A warp works alone.  It owns 4, 8 or 16 rows -- a row is a query token and one of the query heads that share the key/value
// head -- and walks tiles of 32 keys, which it copies itself (cp.async) into a ring of its own in shared memory: nothing
// but the warp's own copies is waited for.  Scores are computed transposed, S^T = K Q^T: 16 keys are the rows of a product's
// left operand, 8 query rows the columns of the right one.  With few query heads per key/value head the other order
// would leave most of a product's 16 rows empty.
//
//   bfloat16 rows     times 2^e, so that a row's largest value is in [2^22, 2^23), and rounded to whole numbers: their three
//                     bytes (the upper one signed) meet the keys' bytes in products of 8-bit integers, whose sums are exact
//                     (at most 255 * 128 * 256 < 2^23 each).  Values down to 2^-15 of the row's largest lose nothing, smaller ones
//                     2^-23 of the largest at most; the keys are used as they lie, without a conversion.
//   float32 rows      times 2^e, the largest in [2^8, 2^9), as a sum of two float16 values (22 bits); keys become float16.
//   int8 -> float16   the byte q + 128 behind the exponent byte 0x64 is the float16 1024 + 128 + q; minus 1152 leaves q
//                     exactly: a byte permutation and a subtraction for two values.
//   values            pairs of dimensions transposed by ldmatrix (two bytes travel as one 16-bit element), so even and odd
//                     dimensions come out as the two halves of a product's 16 rows.
//   scales            u_j = s_kj (k_j . q) scale log2(e) + log2(s_vj) in float32; p'_j = 2^(u_j - M) with M some 2^6 below
//                     the largest u.  O = sum p'_j v8_j, l = sum p'_j / s_vj, and O / l is the result: the value's scale
//                     rides in the exponent, so p' is as large as the term that it stands for.  p' is multiplied as
//                     two float16 parts (what they leave is 2^-22 of itself, or 2^-25 beside a largest of 2^6 and more); l adds
//                     the unrounded.  (Whole-number p' would spare the values' conversion too, but a fixed point takes away the
//                     weights of many faint keys beside a strong one.)
//
// M moves lazily: only when a u has passed it by more than 14 is O rescaled, so most tiles need no reduction over lanes
// at all.
//
// Three forms:
//   attention_8bit_stream   single tokens, long contexts: as many warps as the GPU holds, in teams of a warp for every
//                           key/value head; the tiles of all requests are cut evenly among the teams.  A team's part of a
//                           request is a segment, left in scratch for the merge kernel.
//   attention_8bit_rows     portions, and few or short single tokens: a warp for every 8 or 16 rows, or a block or a
//                           cluster of blocks whose warps share the rows' tiles and meet in shared memory.
//   (bindings)              long bfloat16 portions: pages are widened to 16 bits once (cache_8bit.cu) and read by the
//                           tensor-memory kernel, whose 128-row tiles these 16-row ones cannot match.
//
// What bounds them.  The stream: 64 requests of 3,100 keys on average (205 MB, 31 us at a copy's bandwidth) 44 us: the
// instructions of 16 warps a multiprocessor, how evenly 2,368 of them end, and some 5 us of launch, first tiles and merge.
// (16 / 2 heads of 128, 8 requests of 25,000 keys on average 26.5 us of 16.)  Rows: the matrix instructions and conversions of
// 8 or 16 rows a tile; 2,048 new tokens take 174 us at 32 / 8 heads of 64, widened 47.
#include <cuda_fp16.h>

#include "common.cuh"

#ifndef RV_HD
#define RV_HD 64
#endif
#define A8_HD RV_HD
static_assert(A8_HD % 16 == 0 && A8_HD >= 16 && A8_HD <= 256, "head sizes");
#define A8_KEYS 32                                                // a tile, a lane's key each
#define A8_CHUNKS (A8_HD / 16)                                    // 16-byte pieces of a row
// Warps of a multiprocessor: what the registers (16: 128 a thread, 12: 168, 8: 255) and the rings leave room for.
template <int ROWS, int PARTS> constexpr int a8_warps() {
    constexpr int NT = ROWS > 8 ? 2 : 1;
    return A8_HD <= 64 ? (NT * PARTS == 1 ? 16 : NT * PARTS == 2 ? 12 : 8) : A8_HD <= 192 ? 8 : 6;
}
#define A8_MOST_WARPS 16
#define A8_CLUSTER 8                                              // blocks of a cluster at most
#define A8_BLOCK_WARPS (A8_HD <= 192 ? 4 : 3)

#ifndef A8_STAGES
#define A8_STAGES (A8_HD <= 128 ? 3 : 2)
#endif
#define A8_STAGE_BYTES (2 * A8_KEYS * A8_HD + 2 * A8_KEYS * 4)
#define A8_WARP_BYTES (A8_STAGES * A8_STAGE_BYTES)

struct A8Args {
    const void* q;
    const signed char *k, *v;
    const float *k_scale, *v_scale;
    const int *block_table, *q_start, *ctx_lens;
    const float* sinks;
    void* out;
    float* part_o;                     // [places][rows][HD]
    float2* part_ml;                   // [places][rows]: M, l
    long long q_stride, pages;
    int max_blocks, first_req, n_reqs, num_heads, num_kv_heads, page_size, page_shift, window, nsplit, vec;
    float scale_log2;
};

__device__ __forceinline__ unsigned a8_smem(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void a8_copy16(unsigned dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void a8_copy4(unsigned dst, const void* src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void a8_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                       unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void a8_mma_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0,
                                             unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// int8 times int8 (U: times uint8), sums in int32; 32 terms, or the 16 of a0, a1, b0; `first`: of these alone.
#define A8_IMMA(shape, kind, a_regs, b_regs, ...)                                                                          \
    do {                                                                                                                   \
        if (first)                                                                                                         \
            asm("mma.sync.aligned." shape ".row.col.s32.s8." kind ".s32 {%0,%1,%2,%3}, " a_regs ", " b_regs ", {0,0,0,0};" \
                : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3]) : __VA_ARGS__);                                           \
        else                                                                                                               \
            asm("mma.sync.aligned." shape ".row.col.s32.s8." kind ".s32 {%0,%1,%2,%3}, " a_regs ", " b_regs ", {%0,%1,%2,%3};" \
                : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : __VA_ARGS__);                                           \
    } while (0)
template <bool U>
__device__ __forceinline__ void a8_imma(int (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1,
                                        bool first) {
    if (U) A8_IMMA("m16n8k32", "u8", "{%4,%5,%6,%7}", "{%8,%9}", "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else A8_IMMA("m16n8k32", "s8", "{%4,%5,%6,%7}", "{%8,%9}", "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool U>
__device__ __forceinline__ void a8_imma(int (&c)[4], unsigned a0, unsigned a1, unsigned b0, bool first) {
    if (U) A8_IMMA("m16n8k16", "u8", "{%4,%5}", "{%6}", "r"(a0), "r"(a1), "r"(b0));
    else A8_IMMA("m16n8k16", "s8", "{%4,%5}", "{%6}", "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ unsigned a8_transpose(unsigned x) {
    unsigned y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ unsigned a8_lds(unsigned at) {
    unsigned v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}
__device__ __forceinline__ float a8_max_nan(float a, float b) {       // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float a8_exp2(float x) {              // -inf: 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float a8_pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// Bytes `sel` of x, each behind 0x64, minus 1152 (x: bytes of q + 128).
__device__ __forceinline__ unsigned a8_pair(unsigned x, unsigned sel) {
    const unsigned h = __byte_perm(x, 0x64646464u, sel);
    const __half2 v = __hsub2(*(const __half2*)&h, __half2half2(__ushort_as_half((unsigned short)0x6480)));
    return *(const unsigned*)&v;
}
__device__ __forceinline__ unsigned a8_pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const unsigned*)&h;
}
// What the rounding to float16 left.
__device__ __forceinline__ unsigned a8_rest(float a, float b, unsigned packed) {
    const float2 f = __half22float2(*(const __half2*)&packed);
    return a8_pack(a - f.x, b - f.y);
}
// Where 16-byte piece c of a tile's row lies: moved so that eight rows' pieces c (ldmatrix) are spread over the banks.
__device__ __forceinline__ int a8_piece(int row, int c) {
    constexpr int n = A8_CHUNKS;
    return n % 8 == 0 ? c ^ (row & 7) : n % 4 == 0 ? c ^ ((row >> 1) & 3) : n % 2 == 0 ? c ^ ((row >> 2) & 1) : c;
}

__device__ __forceinline__ float a8_load(const float* p) { return *p; }
__device__ __forceinline__ float a8_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
// N values from p on; `vec`: p is 16-byte aligned.
template <int N>
__device__ __forceinline__ void a8_load_n(const float* p, bool vec, float (&v)[N]) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 f = *(const float4*)(p + i);
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = p[i];
    }
}
template <int N>
__device__ __forceinline__ void a8_load_n(const __nv_bfloat16* p, bool vec, float (&v)[N]) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint2 u = *(const uint2*)(p + i);
            const float2 a = __bfloat1622float2(*(const __nv_bfloat162*)&u.x), b = __bfloat1622float2(*(const __nv_bfloat162*)&u.y);
            v[i] = a.x; v[i + 1] = a.y; v[i + 2] = b.x; v[i + 3] = b.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __bfloat162float(p[i]);
    }
}

// ---- how single tokens' tiles are shared out --------------------------------------------------------
// The tiles of all requests, one after the other, are cut evenly into as many runs as there are teams of warps (`used`
// of them where there are fewer tiles).  A team has a warp for every unit: a key/value head and ROWS of its query
// heads.  Its warps walk the same tiles, so the heads of a page, which lie side by side, are read at about the same time.
// From one segment (a run's part of a request) to the next the run or the request grows, so run + request is a place of
// its own, times the units.
struct A8Shares {
    const int* ctx_lens;
    int n_reqs, window, most;
    long long total, before;           // tiles of all requests; of those before the one asked for
    int used;
    bool narrow;
    static constexpr int KEPT = 4;
    int kept[KEPT];                    // this lane's request's tiles of the first groups of 32 requests
    __device__ __forceinline__ int first(int clen) const { return window > 0 ? max(0, clen - window) / A8_KEYS : 0; }
    // A context that the block table cannot hold has no tiles: the merge marks its rows.
    __device__ __forceinline__ int tiles(int clen) const {
        return clen > 0 && clen <= most ? (clen - 1) / A8_KEYS - first(clen) + 1 : 0;
    }
    __device__ __forceinline__ int length(int r) const { return r < n_reqs ? ctx_lens[r] : 0; }
    // (a whole warp at once)
    __device__ __forceinline__ A8Shares(const int* lens, int reqs, int win, long long slots, int runs, int r)
        : ctx_lens(lens), n_reqs(reqs), window(win), most((int)min(slots, 0x7fffffffll)), total(0), before(0) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int k = 0; k < KEPT; ++k) kept[k] = 32 * k < n_reqs ? length(32 * k + lane) : 0;
#pragma unroll
        for (int k = 0; k < KEPT; ++k) {
            kept[k] = tiles(kept[k]);
            if (32 * k < n_reqs) {
                total += __reduce_add_sync(0xffffffffu, (unsigned)kept[k]);
                if (32 * k < r) before += __reduce_add_sync(0xffffffffu, (unsigned)(32 * k + lane < r ? kept[k] : 0));
            }
        }
        for (int at = 32 * KEPT; at < n_reqs; at += 32) {
            const int mine = tiles(length(at + lane));
            total += __reduce_add_sync(0xffffffffu, (unsigned)mine);
            before += __reduce_add_sync(0xffffffffu, (unsigned)(at + lane < r ? mine : 0));
        }
        used = (int)min((long long)runs, max(1ll, total));
        narrow = total * (used + 1) < 0xffffffffll;
    }
    // (A division of 64 bits takes long enough to be seen.)
    __device__ __forceinline__ long long start(int run) const {
        return narrow ? (long long)((unsigned)run * (unsigned)total / (unsigned)used) : (long long)run * total / used;
    }
    __device__ __forceinline__ int run_of(long long tile) const {
        return narrow ? (int)(((unsigned)(tile + 1) * (unsigned)used - 1u) / (unsigned)total) : (int)(((tile + 1) * used - 1) / total);
    }
};

// ---- one warp's work ----------------------------------------------------------------------------------
// A place in the walk over tiles: the tile `tile` of request r.
struct A8Cursor {
    int r, tile, last, clen;
};

template <typename T, int ROWS, int PARTS>
struct A8Warp {
    static constexpr int NT = ROWS > 8 ? 2 : 1;        // products of 8 columns
    // Four rows take a product's columns twice: what float16 leaves of a weight has the second four, so it costs no product of its own
    // (64 requests of some 3,100 keys, 32 / 8 heads of 64: 44.3 us; as eight rows 46.9).
    static constexpr bool TWICE = ROWS == 4;
    const A8Args& a;
    const unsigned ring;               // in shared memory
    const int lane, g, t;
    int rows_first, rows_count, kvh, G, qs;        // of the segment: its first row, rows, head, query heads a head, first token
    static constexpr bool WHOLE = PARTS == 1;      // queries as whole numbers of 24 bits
    static constexpr int PIECES = WHOLE ? 3 : 2;
    // O^T of 16 dimensions and 8 rows: dimension 2 g (even ones) of rows 2 t, 2 t + 1, then 2 g + 1 of the same
    float o[A8_CHUNKS][NT][4];
    unsigned q[A8_CHUNKS][NT][PIECES];             // WHOLE: upper, middle and lower bytes of 4 values; else 2 and 2, float16
    unsigned q2[WHOLE ? 1 : A8_CHUNKS][NT][2];     // what float16 left of them
    float f[NT][2], M[NT][2], l[NT][2];
    int hi[NT][2], lo[NT][2], p_min, lo_max;

    __device__ __forceinline__ A8Warp(const A8Args& args, unsigned char* mem)
        : a(args), ring(a8_smem(mem)), lane(threadIdx.x & 31), g((threadIdx.x & 31) >> 2), t(threadIdx.x & 3) {
        G = a.num_heads / a.num_kv_heads;
    }

    // The page of this lane's key of a tile (-1: none).  (page_shift: pages of 2^page_shift tokens, or -1.)
    __device__ __forceinline__ int page_of(const A8Cursor& c) const {
        const int key = c.tile * A8_KEYS + lane;
        if (key >= c.clen) return -1;
        const int blk = a.page_shift >= 0 ? key >> a.page_shift : key / a.page_size;
        return blk < a.max_blocks ? a.block_table[(size_t)c.r * a.max_blocks + blk] : -1;
    }
    // A tile's keys and values, piece by piece, and their scales.  In the place of a key without a page comes some row,
    // with scales of 0.
    __device__ __forceinline__ void request(const A8Cursor& c, int head, int page, int stage) const {
        const unsigned base = ring + stage * A8_STAGE_BYTES;
        const int key = c.tile * A8_KEYS + lane;
        const bool ok = page >= 0 && page < a.pages;
        const unsigned block = ok ? (unsigned)page * (unsigned)a.num_kv_heads + (unsigned)head : 0u;
        const int slot = a.page_shift >= 0 ? key & (a.page_size - 1) : key % a.page_size;
        const unsigned row = ok ? block * (unsigned)a.page_size + (unsigned)slot : 0u;
        const unsigned s = base + 2 * A8_KEYS * A8_HD + lane * 4;
        a8_copy4(s, a.k_scale + block, ok);
        a8_copy4(s + A8_KEYS * 4, a.v_scale + block, ok);
        if (a.pages == 0) return;
#pragma unroll
        for (int it = 0; it < A8_CHUNKS; ++it) {                       // 32 keys: a piece a lane each
            const int id = it * 32 + lane, k = id / A8_CHUNKS, c16 = id - k * A8_CHUNKS;
            const size_t at = (size_t)__shfl_sync(0xffffffffu, row, k) * A8_HD + c16 * 16;
            a8_copy16(base + k * A8_HD + a8_piece(k, c16) * 16, a.k + at);
            a8_copy16(base + A8_KEYS * A8_HD + k * A8_HD + a8_piece(k, c16) * 16, a.v + at);
        }
    }

    // Rows [first, first + ROWS) of the `qlen` tokens times G heads of request r.
    __device__ __forceinline__ void begin(int r, int head, int first, int qlen, int q_first, int clen) {
        rows_first = first;
        rows_count = min(ROWS, qlen * G - first);
        kvh = head;
        qs = q_first;
        p_min = clen;
        lo_max = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            // the row whose values this lane holds: column g
            const int i = first + 8 * n + (g & (TWICE ? 3 : 7)), tok = i / G;
            const bool real = i < qlen * G;
            const T* src = (const T*)a.q + (size_t)(qs + (real ? tok : 0)) * a.q_stride +
                           (size_t)(kvh * G + (real ? i - tok * G : 0)) * A8_HD;
            float most = 0.f;
            float x[A8_CHUNKS][4];
#pragma unroll
            for (int c = 0; c < A8_CHUNKS; ++c) a8_load_n<4>(src + 16 * c + 4 * t, a.vec, x[c]);
#pragma unroll
            for (int c = 0; c < A8_CHUNKS; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (!real) x[c][k] = 0.f;
                    most = a8_max_nan(most, fabsf(x[c][k]));
                }
            most = a8_max_nan(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = a8_max_nan(most, __shfl_xor_sync(0xffffffffu, most, 2));
            // the largest in [2^22, 2^23), or in [2^8, 2^9): times 2^e, e between -120 and 149, as two factors that float32
            // holds (a row's values may be of any size)
            const int e = most > 0.f ? (WHOLE ? 22 : 8) - ((int)(__float_as_uint(most) >> 23) - 127) : 0;     // (NaN: 0)
            const int e1 = e / 2, e2 = e - e1;
            const float up1 = a8_pow2(e1), up2 = a8_pow2(e2);
            float mine = a.scale_log2 * a8_pow2(-e1) * a8_pow2(-e2);
            if (WHOLE && !(most <= 3.402823466e38f)) mine = NAN;       // whole numbers hold no infinity
#pragma unroll
            for (int c = 0; c < A8_CHUNKS; ++c) {
                if constexpr (WHOLE) {
#pragma unroll
                    for (int p = 0; p < PIECES; ++p) q[c][n][p] = 0u;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int v = __float2int_rn(x[c][k] * up1 * up2);        // (bfloat16: at most 255 * 2^15)
#pragma unroll
                        for (int p = 0; p < PIECES; ++p) q[c][n][p] |= ((unsigned)(v >> (16 - 8 * p)) & 0xffu) << (8 * k);
                    }
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float x0 = x[c][2 * h] * up1 * up2, x1 = x[c][2 * h + 1] * up1 * up2;
                        q[c][n][h] = a8_pack(x0, x1);
                        q2[c][n][h] = a8_rest(x0, x1, q[c][n][h]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // the rows of this lane's scores: columns 2 t, 2 t + 1
                f[n][h] = __shfl_sync(0xffffffffu, mine, (2 * t + h) * 4);
                const int j = first + 8 * n + ((2 * t + h) & (TWICE ? 3 : 7));
                hi[n][h] = j < qlen * G ? clen - qlen + j / G : -1;
                lo[n][h] = a.window > 0 ? max(0, hi[n][h] - a.window + 1) : 0;
                M[n][h] = -INFINITY;
                l[n][h] = 0.f;
            }
        }
        // rows come in the order of their tokens
        p_min = clen - qlen + first / G;
        const int p_max = clen - qlen + (first + rows_count - 1) / G;
        lo_max = a.window > 0 ? max(0, p_max - a.window + 1) : 0;
#pragma unroll
        for (int c = 0; c < A8_CHUNKS; ++c)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[c][n][k] = 0.f;
    }

    // S^T of 16 keys as float32.
    __device__ __forceinline__ void scores(unsigned base, int m, float (&s)[NT][4]) {
        // pieces c and c + 1 of the 16 keys' rows: lanes 0-7, 8-15 name keys 0-7, 8-15 of piece c, the others of c + 1
        const int key = 16 * m + (lane & 15);
        int up[NT][4], mid[NT][4], low[NT][4];
        auto half = [&](int c, unsigned w0, unsigned w1) {            // 16 dimensions, float16
            w0 ^= 0x80808080u;
            w1 ^= 0x80808080u;
            const unsigned a0 = a8_pair(w0, 0x4140), a2 = a8_pair(w0, 0x4342);
            const unsigned a1 = a8_pair(w1, 0x4140), a3 = a8_pair(w1, 0x4342);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (c == 0) a8_mma_first(s[n], a0, a1, a2, a3, q[c][n][0], q[c][n][1]);
                else a8_mma(s[n], a0, a1, a2, a3, q[c][n][0], q[c][n][1]);
                a8_mma(s[n], a0, a1, a2, a3, q2[WHOLE ? 0 : c][n][0], q2[WHOLE ? 0 : c][n][1]);
            }
        };
#pragma unroll
        for (int c = 0; c < A8_CHUNKS; c += 2) {
            unsigned w[4];
            if (c + 1 < A8_CHUNKS) {
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(base + key * A8_HD + a8_piece(key, c + (lane >> 4)) * 16));
                if constexpr (WHOLE) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        a8_imma<false>(up[n], w[0], w[1], w[2], w[3], q[c][n][0], q[c + 1 < A8_CHUNKS ? c + 1 : c][n][0], c == 0);
                        a8_imma<true>(mid[n], w[0], w[1], w[2], w[3], q[c][n][1], q[c + 1 < A8_CHUNKS ? c + 1 : c][n][1], c == 0);
                        a8_imma<true>(low[n], w[0], w[1], w[2], w[3], q[c][n][PIECES - 1], q[c + 1 < A8_CHUNKS ? c + 1 : c][n][PIECES - 1], c == 0);
                    }
                } else {
                    half(c, w[0], w[1]);
                    half(c + 1, w[2], w[3]);
                }
            } else {
                asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];"
                             : "=r"(w[0]), "=r"(w[1]) : "r"(base + key * A8_HD + a8_piece(key, c) * 16));
                if constexpr (WHOLE) {
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        a8_imma<false>(up[n], w[0], w[1], q[c][n][0], c == 0);
                        a8_imma<true>(mid[n], w[0], w[1], q[c][n][1], c == 0);
                        a8_imma<true>(low[n], w[0], w[1], q[c][n][PIECES - 1], c == 0);
                    }
                } else {
                    half(c, w[0], w[1]);
                }
            }
        }
        if constexpr (WHOLE) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) s[n][k] = fmaf((float)(up[n][k] * 256 + mid[n][k]), 256.f, (float)low[n][k]);
        }
    }

    // The rows' references to x, which are larger: O and l follow.
    __device__ __forceinline__ void move(int n, int j, float x) {
        const float corr = x == -INFINITY ? 1.f : a8_exp2(M[n][j] - x);                 // M = -inf: 0
        M[n][j] = x;
        l[n][j] *= corr;
#pragma unroll
        for (int c = 0; c < A8_CHUNKS; ++c)
#pragma unroll
            for (int k = j; k < 4; k += 2) o[c][n][k] *= corr;
    }
    __device__ __forceinline__ void tile(int tile_at, int stage) {
        const unsigned base = ring + stage * A8_STAGE_BYTES, scales = base + 2 * A8_KEYS * A8_HD + 4 * lane;
        constexpr int MT = A8_KEYS / 16;
        float s[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; ++m) scores(base, m, s[m]);
        // ---- u, its largest -------------------------------------------------------------------------
        const int key0 = tile_at * A8_KEYS;
        // this lane's key: its scale, log2 of its value's scale and one over that; a key without a page (its scales
        // are zeros) shows in every row that may see it
        const float sk1 = __uint_as_float(a8_lds(scales));
        const int e1 = max(-60, min(60, (int)((a8_lds(scales + 4 * A8_KEYS) >> 23) & 0xff) - 127));
        const float inv1 = __uint_as_float((unsigned)(127 - e1) << 23), ev1 = sk1 == 0.f ? NAN : (float)e1;
        float inv[MT][2], mx[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) mx[n][0] = mx[n][1] = -INFINITY;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = 16 * m + 8 * h + g;
                const float sk = __shfl_sync(0xffffffffu, sk1, key), ev = __shfl_sync(0xffffffffu, ev1, key);
                inv[m][h] = __shfl_sync(0xffffffffu, inv1, key);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int j = 0; j < 2; ++j) s[m][n][2 * h + j] = fmaf(s[m][n][2 * h + j], f[n][j] * sk, ev);
            }
        if (key0 + A8_KEYS - 1 > p_min || key0 < lo_max) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int key = key0 + 16 * m + 8 * h + g;
                            if (key > hi[n][j] || key < lo[n][j]) s[m][n][2 * h + j] = -INFINITY;
                        }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) mx[n][j] = fmaxf(mx[n][j], fmaxf(s[m][n][j], s[m][n][2 + j]));
        // p' is at most 2^6 when its reference is set and may grow to 2^14
        bool moves = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) moves |= mx[n][j] > M[n][j] + 14.f;           // also from -inf
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float x = mx[n][j];
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                    move(n, j, fmaxf(x - 6.f, M[n][j]));
                }
        }
        // ---- p', l, and O^T += V^T P^T ----------------------------------------------------------------
        float off[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) off[n][j] = M[n][j] == -INFINITY ? 0.f : M[n][j];
        const unsigned vbase = base + A8_KEYS * A8_HD;
        unsigned p[NT][MT][2], p2[NT][MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p0 = a8_exp2(s[m][n][2 * h] - off[n][0]), p1 = a8_exp2(s[m][n][2 * h + 1] - off[n][1]);
                    l[n][0] = fmaf(p0, inv[m][h], l[n][0]);
                    l[n][1] = fmaf(p1, inv[m][h], l[n][1]);
                    const unsigned w = a8_pack(p0, p1);
                    const unsigned rest = a8_rest(p0, p1, w);
                    p[n][m][h] = a8_transpose(TWICE && t >= 2 ? rest : w);
                    if (!TWICE) p2[n][m][h] = a8_transpose(rest);
                }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            // pieces c and c + 1 of the 16 keys' rows: lanes 0-7, 8-15 name keys 0-7, 8-15 of piece c, the others of c + 1
            const int key = 16 * m + (lane & 15);
#pragma unroll
            for (int c = 0; c < A8_CHUNKS; c += 2) {
                unsigned w[4];
                if (c + 1 < A8_CHUNKS) {
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                                 : "r"(vbase + key * A8_HD + a8_piece(key, c + (lane >> 4)) * 16));
                } else {
                    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];"
                                 : "=r"(w[0]), "=r"(w[1])
                                 : "r"(vbase + key * A8_HD + a8_piece(key, c) * 16));
                    w[2] = w[3] = 0u;
                }
#pragma unroll
                for (int k = 0; k < 2 && c + k < A8_CHUNKS; ++k) {
                    const unsigned x = w[2 * k] ^ 0x80808080u, y = w[2 * k + 1] ^ 0x80808080u;
                    const unsigned a0 = a8_pair(x, 0x4240), a1 = a8_pair(x, 0x4341);
                    const unsigned a2 = a8_pair(y, 0x4240), a3 = a8_pair(y, 0x4341);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        a8_mma(o[c + k][n], a0, a1, a2, a3, p[n][m][0], p[n][m][1]);
                        if (!TWICE) a8_mma(o[c + k][n], a0, a1, a2, a3, p2[n][m][0], p2[n][m][1]);
                    }
                }
            }
        }
    }
    // Sums over the lanes that share a row.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 4);
                l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 8);
                l[n][j] += __shfl_xor_sync(0xffffffffu, l[n][j], 16);
            }
        if (TWICE)
#pragma unroll
            for (int c = 0; c < A8_CHUNKS; ++c)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[c][0][k] += __shfl_xor_sync(0xffffffffu, o[c][0][k], 2);
    }
    __device__ __forceinline__ void leave(size_t place) {
        finish();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = 8 * n + 2 * t + j;
                if (row >= rows_count) continue;
                const size_t at = place * ROWS + row;
                if (g == 0) a.part_ml[at] = make_float2(M[n][j], l[n][j]);
#pragma unroll
                for (int c = 0; c < A8_CHUNKS; ++c)
                    *(float2*)(a.part_o + at * A8_HD + 16 * c + 2 * g) = make_float2(o[c][n][j], o[c][n][2 + j]);
            }
    }
};

#define A8_WAIT_STAGE() asm volatile("cp.async.wait_group %0;" ::"n"(A8_STAGES - 2) : "memory")
#define A8_COMMIT() asm volatile("cp.async.commit_group;" ::: "memory")

// Requests [0, n_reqs) with one token each.
template <typename T, int ROWS, int PARTS>
__global__ void __launch_bounds__(A8_BLOCK_WARPS * 32, a8_warps<ROWS, PARTS>() / A8_BLOCK_WARPS) attention_8bit_stream_kernel(const __grid_constant__ A8Args a) {
    rv_pdl_wait();
    rv_pdl_launch_dependents();        // the merge may read what was there before this launch as soon as it begins
    extern __shared__ __align__(128) unsigned char smem[];
    A8Warp<T, ROWS, PARTS> w(a, smem + (threadIdx.x >> 5) * A8_WARP_BYTES);
    const int per_head = (w.G + ROWS - 1) / ROWS, units = a.num_kv_heads * per_head;
    const int warps = gridDim.x * A8_BLOCK_WARPS, teams = max(1, warps / units);
    const A8Shares sh(a.ctx_lens, a.n_reqs, a.window, (long long)a.max_blocks * a.page_size, teams, 0);
    if (sh.total == 0) return;
    // (more units than warps: a warp has several of the one team's)
    for (int slot = blockIdx.x * A8_BLOCK_WARPS + (threadIdx.x >> 5); slot < teams * units; slot += warps) {
        const int run = slot / units, u = slot - run * units, head = u / per_head;
        if (run >= sh.used) return;
        const long long from = sh.start(run);
        const int n = (int)(sh.start(run + 1) - from);
        // where the run begins
        A8Cursor c = {0, 0, 0, 0};
        {
            const int lane = threadIdx.x & 31;
            long long sum = 0;
            bool found = false;
            auto look = [&](int at, int mine) {
                int upto = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= d) upto += v;
                }
                const unsigned who = __ballot_sync(0xffffffffu, sum + upto > from);
                if (who) {
                    const int l = __ffs(who) - 1;
                    c.r = at + l;
                    c.clen = sh.length(c.r);
                    c.tile = sh.first(c.clen) + (int)(from - sum) - __shfl_sync(0xffffffffu, upto - mine, l);
                    c.last = (c.clen - 1) / A8_KEYS;
                    found = true;
                }
                sum += __shfl_sync(0xffffffffu, upto, 31);
            };
#pragma unroll
            for (int k = 0; k < A8Shares::KEPT; ++k)
                if (!found && 32 * k < a.n_reqs) look(32 * k, sh.kept[k]);
            for (int at = 32 * A8Shares::KEPT; !found && at < a.n_reqs; at += 32) look(at, sh.tiles(sh.length(at + lane)));
        }
        auto advance = [&](A8Cursor& x) {
            if (++x.tile <= x.last) return;
            do ++x.r;
            while (x.r < a.n_reqs && sh.tiles(sh.length(x.r)) == 0);
            x.clen = sh.length(x.r);
            x.last = (x.clen - 1) / A8_KEYS;
            x.tile = sh.first(x.clen);
        };
        A8Cursor ahead = c;
        int page = w.page_of(ahead), requested = 0;
        auto request_next = [&](int stage) {
            if (requested < n) {
                w.request(ahead, head, page, stage);
                if (++requested < n) {
                    advance(ahead);
                    page = w.page_of(ahead);
                }
            }
            A8_COMMIT();
        };
        for (int i = 0; i < A8_STAGES - 1; ++i) request_next(i);
        bool fresh = true;
        int stage = 0;
        for (int i = 0; i < n; ++i) {
            if (fresh) {
                w.begin(c.r, head, (u - head * per_head) * ROWS, 1, c.r, c.clen);
                fresh = false;
            }
            A8_WAIT_STAGE();
            __syncwarp();
            request_next(stage == 0 ? A8_STAGES - 1 : stage - 1);
            w.tile(c.tile, stage);
            __syncwarp();
            stage = stage + 1 == A8_STAGES ? 0 : stage + 1;
            if (c.tile == c.last || i + 1 == n) {
                w.leave(((size_t)run + c.r) * units + u);
                fresh = true;
            }
            if (i + 1 < n) advance(c);
        }
    }
}

// ---- rows whose tiles a warp, a block or a cluster of blocks has ---------------------------------------------
__device__ __forceinline__ unsigned a8_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void a8_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 a8_remote(const void* p, int rank) {
    unsigned at;
    float2 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(a8_smem(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
// What N parts of a row come to: their M and l (ml) and two of their dimensions.  A part with l = 0 weighs nothing.
template <int N>
__device__ __forceinline__ void a8_join(const float2 (&ml)[N], const float2 (&v)[N], float2& all, float2& o) {
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) M = fmaxf(M, ml[i].x);
    const float off = M == -INFINITY ? 0.f : M;
    all = make_float2(M, 0.f);
    o = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float w = a8_exp2(ml[i].x - off);
        all.y += ml[i].x == -INFINITY ? ml[i].y : ml[i].y * w;        // (without a reference: 0, or not a number)
        o.x = fmaf(v[i].x, w, o.x);
        o.y = fmaf(v[i].y, w, o.y);
    }
}
template <typename T>
__device__ __forceinline__ void a8_put(const A8Args& a, int row_token, int head, int dim, float2 all, float2 o) {
    float L = all.y;
    if (a.sinks && L != 0.f) L += a8_exp2(a.sinks[head] * 1.4426950408889634f - all.x);       // a sink counts once
    const float by = L == 0.f ? 0.f : 1.f / L;
    T* dst = (T*)a.out + ((size_t)row_token * a.num_heads + head) * A8_HD + dim;
    rv_store(dst, o.x * by);
    rv_store(dst + 1, o.y * by);
}

// Requests [first_req, first_req + n_reqs) with any number of tokens.  blockIdx.z: request, y: key/value head, x: ROWS rows
// a warp (nsplit 0), or a cluster of nsplit blocks: their warps share the rows' tiles and meet in the blocks'
// shared memory, then in the cluster's.
template <typename T, int ROWS, int PARTS, bool SHARED>
__global__ void __launch_bounds__(A8_BLOCK_WARPS * 32, a8_warps<ROWS, PARTS>() / A8_BLOCK_WARPS) attention_8bit_rows_kernel(
    const __grid_constant__ A8Args a) {
    rv_pdl_prologue();
    constexpr int NT = ROWS > 8 ? 2 : 1;
    extern __shared__ __align__(128) unsigned char smem[];
    const int warp = threadIdx.x >> 5, rank = SHARED && a.nsplit > 1 ? (int)a8_rank() : 0;
    const int rt = SHARED ? blockIdx.x / a.nsplit : blockIdx.x * A8_BLOCK_WARPS + warp;
    const int parts = SHARED ? a.nsplit * A8_BLOCK_WARPS : 1, part = SHARED ? rank * A8_BLOCK_WARPS + warp : 0;
    const int r = a.first_req + blockIdx.z, head = blockIdx.y;
    const int qs = a.q_start[r], qlen = a.q_start[r + 1] - qs, clen = a.ctx_lens[r];
    A8Warp<T, ROWS, PARTS> w(a, smem + warp * A8_WARP_BYTES);
    // the rows with the longest contexts first
    const int tiles = (qlen * w.G + ROWS - 1) / ROWS;
    if (rt >= tiles) return;                                           // (a whole cluster)
    const int first = (tiles - 1 - rt) * ROWS;
    const int end = min(qlen * w.G, first + ROWS);
    const int p_first = clen - qlen + first / w.G, p_last = clen - qlen + (end - 1) / w.G;
    const bool fits = clen <= (long long)a.max_blocks * a.page_size;
    const int t_all = (a.window > 0 ? max(0, p_first - a.window + 1) : 0) / A8_KEYS;
    const int count = p_last >= 0 && fits ? p_last / A8_KEYS - t_all + 1 : 0;
    const int t_lo = t_all + (int)((long long)count * part / parts), n = t_all + (int)((long long)count * (part + 1) / parts) - t_lo;
    A8Cursor ahead = {r, t_lo, t_lo + n - 1, clen};
    int page = n > 0 ? w.page_of(ahead) : -1, requested = 0;
    auto request_next = [&](int stage) {
        if (requested < n) {
            w.request(ahead, head, page, stage);
            ++ahead.tile;
            if (++requested < n) page = w.page_of(ahead);
        }
        A8_COMMIT();
    };
    for (int i = 0; i < A8_STAGES - 1; ++i) request_next(i);
    w.begin(r, head, first, qlen, qs, clen);
    int stage = 0;
    for (int i = 0; i < n; ++i) {
        A8_WAIT_STAGE();
        __syncwarp();
        request_next(stage == 0 ? A8_STAGES - 1 : stage - 1);
        w.tile(t_lo + i, stage);
        __syncwarp();
        stage = stage + 1 == A8_STAGES ? 0 : stage + 1;
    }
    if (!fits) {
#pragma unroll
        for (int k = 0; k < NT; ++k) w.l[k][0] = w.l[k][1] = NAN;      // more keys than the table holds
    }
    w.finish();
    if constexpr (!SHARED) {
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int i = first + 8 * k + 2 * w.t + j, tok = i / w.G;
                if (i < end)
#pragma unroll
                    for (int c = 0; c < A8_CHUNKS; ++c)
                        a8_put<T>(a, qs + tok, head * w.G + i - tok * w.G, 16 * c + 2 * w.g, make_float2(w.M[k][j], w.l[k][j]),
                                  make_float2(w.o[c][k][j], w.o[c][k][2 + j]));
            }
    } else {
        // [row][HD + 8] of a warp, in the place of its ring (every copy into it has been waited for)
        constexpr int STRIDE = A8_HD + 8;
        static_assert(8 * NT * STRIDE * 4 <= A8_WARP_BYTES, "a warp's rows fit its ring");
        __shared__ float2 ml[A8_BLOCK_WARPS][8 * NT], ml_block[8 * NT];
        float* rows_of = (float*)(smem + warp * A8_WARP_BYTES);
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = 8 * k + 2 * w.t + j;
                if (w.g == 0) ml[warp][row] = make_float2(w.M[k][j], w.l[k][j]);
#pragma unroll
                for (int c = 0; c < A8_CHUNKS; ++c)
                    *(float2*)(rows_of + row * STRIDE + 16 * c + 2 * w.g) = make_float2(w.o[c][k][j], w.o[c][k][2 + j]);
            }
        __syncthreads();
        const int rows = end - first;
        for (int i = threadIdx.x; i < rows * (A8_HD / 2); i += A8_BLOCK_WARPS * 32) {
            const int row = i / (A8_HD / 2), dim = (i - row * (A8_HD / 2)) * 2, at = row * STRIDE + dim;
            float2 m[A8_BLOCK_WARPS], v[A8_BLOCK_WARPS], all, o;
#pragma unroll
            for (int k = 0; k < A8_BLOCK_WARPS; ++k) {
                m[k] = ml[k][row];
                v[k] = *(const float2*)((const float*)(smem + k * A8_WARP_BYTES) + at);
            }
            a8_join(m, v, all, o);
            if (a.nsplit == 1) {
                const int x = first + row, tok = x / w.G;
                a8_put<T>(a, qs + tok, head * w.G + x - tok * w.G, dim, all, o);
            } else {
                *(float2*)((float*)smem + at) = o;                     // nobody else's
                if (dim == 0) ml_block[row] = all;
            }
        }
        if (a.nsplit == 1) return;
        a8_cluster_sync();
        for (int i = rank * A8_BLOCK_WARPS * 32 + threadIdx.x; i < rows * (A8_HD / 2); i += a.nsplit * A8_BLOCK_WARPS * 32) {
            const int row = i / (A8_HD / 2), dim = (i - row * (A8_HD / 2)) * 2, at = row * STRIDE + dim;
            float2 m[A8_CLUSTER], v[A8_CLUSTER], all, o;
#pragma unroll
            for (int k = 0; k < A8_CLUSTER; ++k) {
                m[k] = make_float2(-INFINITY, 0.f);
                v[k] = make_float2(0.f, 0.f);
                if (k < a.nsplit) {
                    m[k] = a8_remote(&ml_block[row], k);
                    v[k] = a8_remote((const float*)smem + at, k);
                }
            }
            a8_join(m, v, all, o);
            const int x = first + row, tok = x / w.G;
            a8_put<T>(a, qs + tok, head * w.G + x - tok * w.G, dim, all, o);
        }
        a8_cluster_sync();                                             // nobody leaves while its rows are read
    }
}

// ---- segments put together, in order --------------------------------------------------------------------
// `W` warps a row, which share its segments (eight where there may be many; a lane has two of every 64 dimensions and
// requests eight segments' before it uses any: one memory latency for eight).
template <typename T, int W>
__device__ __forceinline__ void a8_merge(const A8Args& a, size_t place, int n, int units, int rows, int row, int head, T* dst, bool bad) {
    const size_t step = (size_t)units * rows, at0 = place * rows + row;           // of a place's row to the next run's
    const int lane = threadIdx.x & 31, part = W == 1 ? 0 : threadIdx.x >> 5;
    constexpr int PER = (A8_HD + 63) / 64, AHEAD = 8;
    float2 o[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) o[k] = make_float2(0.f, 0.f);
    float M = -INFINITY, L = 0.f;
    for (int at = part * AHEAD; at < n; at += W * AHEAD) {
        const float2 ml = lane < AHEAD && at + lane < n ? a.part_ml[at0 + (at + lane) * step] : make_float2(-INFINITY, 0.f);
        float2 v[AHEAD][PER];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
#pragma unroll
            for (int k = 0; k < PER; ++k)
                v[i][k] = at + i < n && (A8_HD % 64 == 0 || 64 * k + 2 * lane < A8_HD)
                              ? *(const float2*)(a.part_o + (at0 + (at + i) * step) * A8_HD + 64 * k + 2 * lane)
                              : make_float2(0.f, 0.f);
        const float most = fmaxf(M, rv_warp_max(ml.x));
        const float off = most == -INFINITY ? 0.f : most;
        const float keep = a8_exp2(M - off), w = a8_exp2(ml.x - off);
        L = L * keep + rv_warp_sum(ml.x == -INFINITY ? ml.y : ml.y * w);      // (without a reference: 0, or not a number)
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            o[k].x *= keep;
            o[k].y *= keep;
        }
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float wi = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                o[k].x = fmaf(v[i][k].x, wi, o[k].x);
                o[k].y = fmaf(v[i][k].y, wi, o[k].y);
            }
        }
        M = most;
    }
    if (W > 1) {
        __shared__ float2 rows[W][PER * 32], ml[W];
        if (lane == 0) ml[part] = make_float2(M, L);
#pragma unroll
        for (int k = 0; k < PER; ++k) rows[part][32 * k + lane] = o[k];
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int i = 0; i < W; ++i) M = fmaxf(M, ml[i].x);
        const float off = M == -INFINITY ? 0.f : M;
        L = 0.f;
#pragma unroll
        for (int k = 0; k < PER; ++k) o[k] = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float w = a8_exp2(ml[i].x - off);
            L += ml[i].x == -INFINITY ? ml[i].y : ml[i].y * w;
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                o[k].x = fmaf(rows[i][32 * k + lane].x, w, o[k].x);
                o[k].y = fmaf(rows[i][32 * k + lane].y, w, o[k].y);
            }
        }
    }
    if (a.sinks && L != 0.f) L += a8_exp2(a.sinks[head] * 1.4426950408889634f - M);
    const float by = bad ? NAN : L == 0.f ? 0.f : 1.f / L;
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (64 * k + 2 * lane < A8_HD) {
            rv_store(dst + 64 * k + 2 * lane, bad ? NAN : o[k].x * by);
            rv_store(dst + 64 * k + 2 * lane + 1, bad ? NAN : o[k].y * by);
        }
}

// A warp (W = 1: four rows a block) or a block a row; blockIdx.y: request, x: head.  It lets no launch behind it begin
// before it is done: blocks of the next stream that wait where this one's have yet to run cost 17 us of 60 a call.
template <typename T, int ROWS, int W>
__global__ void __launch_bounds__(W == 1 ? 128 : W * 32) attention_8bit_stream_merge_kernel(const __grid_constant__ A8Args a, int runs) {
    const int G = a.num_heads / a.num_kv_heads, per_head = (G + ROWS - 1) / ROWS, units = a.num_kv_heads * per_head;
    const int r = blockIdx.y, head = W == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
    if (head >= a.num_heads) {
        rv_pdl_wait();
        return;
    }
    const int kvh = head / G, in = head - kvh * G, u = kvh * per_head + in / ROWS;
    const A8Shares sh(a.ctx_lens, a.n_reqs, a.window, (long long)a.max_blocks * a.page_size, runs, r);
    const int clen = sh.length(r), tiles = sh.tiles(clen);
    int run0 = 0, n = 0;
    if (tiles) {
        run0 = sh.run_of(sh.before);
        n = sh.run_of(sh.before + tiles - 1) - run0 + 1;
    }
    rv_pdl_wait();
    a8_merge<T, W>(a, ((size_t)run0 + r) * units + u, n, units, ROWS, in % ROWS, head,
                   (T*)a.out + ((size_t)r * a.num_heads + head) * A8_HD, clen > 0 && tiles == 0);
}

// ---- host side ----------------------------------------------------------------------------------------
static thread_local char g_a8_error[512] = "";
#define A8_FAIL(...) do { snprintf(g_a8_error, sizeof(g_a8_error), __VA_ARGS__); return 1; } while (0)
#define A8_CAT2(x, y) x##y
#define A8_CAT(x, y) A8_CAT2(x, y)
#define A8_SYM(name) A8_CAT(A8_CAT(name, _hd), RV_HD)

extern "C" const char* A8_SYM(rv_attention_8bit_last_error)() { return g_a8_error; }

// Rows of a warp: 16 where a key/value head has more than 8 of them and the accumulators fit the registers, 4 where it has no more.
static int a8_row_count(long long rows) { return rows <= 4 ? 4 : rows > 8 && A8_HD <= 128 ? 16 : 8; }
static long long a8_place_bytes(int rows) { return (long long)rows * (A8_HD * 4 + 8); }

static long long a8_tiles(int max_ctx_len, int window, int max_q_len) {
    long long keys = max_ctx_len;
    if (window > 0 && (long long)window + max_q_len < keys) keys = (long long)window + max_q_len;
    return (keys + A8_KEYS - 1) / A8_KEYS;
}
// Blocks whose warps share the tiles of ROWS rows: 0 (a warp has them alone) where there are warps enough, else as many as the
// GPU holds at once, up to a cluster, while every warp has a tile.  (us by warps alone / a block / two / four / eight: 32 / 8
// heads of 64, 128 requests of 700 keys 35 / 23 / 34 / 53 / 84, 32 of 1,000 24 / 15 / 11.8 / 16 / 25, 16 of 4,000 78 / 30 / 26 / 17 / 22.)
static int a8_nsplit(long long units, long long tiles, int block_places) {
    if (units > 4ll * block_places || tiles < 2) return 0;
    int n = 1;
    while (2 * n <= A8_CLUSTER && units * 2 * n <= block_places && tiles >= 2ll * n * A8_BLOCK_WARPS) n *= 2;
    return n;
}
// Single tokens by blocks or clusters, which need no scratch and no second launch, but take as long as the longest context: while
// a warp has no more than eight tiles of that, in two rounds at most.  (us so / by the stream: 32 / 8 heads of 64, 1 request of
// 700 keys 5.2 / 6.0, 64 of 100 7.4 / 10.6, 64 of 700 12.6 / 17.6, 128 of 700 23.6 / 26.3, 16 of 4,000 16.9 / 19.9; 8 / 8 heads of
// 128, 32 of 1,000 13.8 / 17.6, 128 of 300 (1,024 blocks for 296 places) 25 / 22; 16 / 2 heads of 128, 8 of 31,000 43 / 30.  Near the
// border, 64 of 2,000 alike 28 / 33, of 2,340 to 3,850 43 / 44.)
static bool a8_few(long long units, long long tiles, int n_sms, int form) {
    if (form != 0) return form == 2;               // 1: the stream, 2: blocks and clusters
    const int places = (A8_HD <= 64 ? 4 : 2) * n_sms;
    const int n = a8_nsplit(units, tiles, places);
    return units <= 2ll * places && tiles <= 8ll * A8_BLOCK_WARPS * (n ? n : 1);
}

// Scratch for single tokens: requests [0, n_decode).
extern "C" long long A8_SYM(rv_paged_attention_8bit_scratch_bytes)(int n_decode, int max_ctx_len, int num_heads, int num_kv_heads,
                                                                   int window, int n_sms, int form) {
    const int G = num_heads / num_kv_heads, rows = a8_row_count(G);
    const long long units = (long long)num_kv_heads * ((G + rows - 1) / rows);
    if (n_decode <= 0 || a8_few(units * n_decode, a8_tiles(max_ctx_len, window, 1), n_sms, form)) return 0;
    const long long all = (long long)n_sms * A8_MOST_WARPS;
    return ((all > units ? all : units) + n_decode * units) * a8_place_bytes(rows);
}

// The limit of shared memory is a kernel's on a device: raised once on each.
#define A8_CONFIGURE(kernel, smem)                                                                              \
    do {                                                                                                        \
        static bool done[64];                                                                                   \
        int dev = 0;                                                                                            \
        if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) A8_FAIL("paged_attention_8bit: no device"); \
        if (!done[dev]) {                                                                                       \
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(smem)); \
            if (e != cudaSuccess) A8_FAIL("paged_attention_8bit: %s", cudaGetErrorString(e));                   \
            done[dev] = true;                                                                                   \
        }                                                                                                       \
    } while (0)

template <typename T, int ROWS, int PARTS>
static int a8_stream(A8Args a, int n_sms, cudaStream_t stream) {
    const size_t smem = (size_t)A8_BLOCK_WARPS * A8_WARP_BYTES;
    const int blocks = n_sms * (a8_warps<ROWS, PARTS>() / A8_BLOCK_WARPS);
    auto kernel = attention_8bit_stream_kernel<T, ROWS, PARTS>;
    A8_CONFIGURE(kernel, smem);
    const int G = a.num_heads / a.num_kv_heads;
    const long long per = a.num_kv_heads * ((G + ROWS - 1) / ROWS), all = (long long)blocks * A8_BLOCK_WARPS;
    const long long places = (all > per ? all : per) + a.n_reqs * per;
    a.part_ml = (float2*)(a.part_o + places * ROWS * A8_HD);
    rv_launch(kernel, dim3(blocks), dim3(A8_BLOCK_WARPS * 32), smem, stream, a);
    // segments of a request, about: runs a request
    const int units = a.num_kv_heads * ((G + ROWS - 1) / ROWS), warps = blocks * A8_BLOCK_WARPS;
    const int teams = warps / units > 1 ? warps / units : 1;
    if (teams > 8 * a.n_reqs)
        rv_launch(attention_8bit_stream_merge_kernel<T, ROWS, 8>, dim3(a.num_heads, a.n_reqs), dim3(256), 0, stream, a, teams);
    else
        rv_launch(attention_8bit_stream_merge_kernel<T, ROWS, 1>, dim3((a.num_heads + 3) / 4, a.n_reqs), dim3(128), 0, stream, a, teams);
    return 0;
}
// `tokens`, `depth`: about how many tokens the requests bring in all, and how deep they are.  Which form is chosen follows these; the
// launch's size follows the longest.
template <typename T, int ROWS, int PARTS>
static int a8_rows(A8Args a, long long tokens, int max_q_len, int depth, int n_sms, cudaStream_t stream) {
    const size_t smem = (size_t)A8_BLOCK_WARPS * A8_WARP_BYTES;
    const long long rows = (long long)max_q_len * (a.num_heads / a.num_kv_heads);
    if (rows > 0x7fffffffll) A8_FAIL("paged_attention_8bit: too many rows");
    const int row_tiles = (int)((rows + ROWS - 1) / ROWS);
    // (a padded step launches blocks for every request as if it were the longest, most of which find no rows: of one portion of 64
    // tokens after 1,000 beside an empty one 17.8 us by what is launched, 14.6 by what is there)
    const long long there = tokens * (a.num_heads / a.num_kv_heads) / ROWS + a.n_reqs, launched = (long long)row_tiles * a.n_reqs;
    a.nsplit = a8_nsplit((there < launched ? there : launched) * a.num_kv_heads, a8_tiles(depth, a.window, max_q_len),
                         n_sms * (a8_warps<ROWS, PARTS>() / A8_BLOCK_WARPS));
    if (a.nsplit == 0) {
        auto kernel = attention_8bit_rows_kernel<T, ROWS, PARTS, false>;
        A8_CONFIGURE(kernel, smem);
        rv_launch(kernel, dim3((unsigned)((row_tiles + A8_BLOCK_WARPS - 1) / A8_BLOCK_WARPS), a.num_kv_heads, a.n_reqs),
                  dim3(A8_BLOCK_WARPS * 32), smem, stream, a);
        return 0;
    }
    auto kernel = attention_8bit_rows_kernel<T, ROWS, PARTS, true>;
    A8_CONFIGURE(kernel, smem);
    if ((long long)row_tiles * a.nsplit > 0x7fffffffll) A8_FAIL("paged_attention_8bit: too many rows");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(row_tiles * a.nsplit), a.num_kv_heads, a.n_reqs);
    cfg.blockDim = dim3(A8_BLOCK_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = rv_pdl_enabled();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.nsplit;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.nsplit > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) A8_FAIL("paged_attention_8bit: %s", cudaGetErrorString(e));
    return 0;
}
template <typename T, int PARTS>
static int a8_portions(const A8Args& a, long long tokens, int max_q_len, int depth, int n_sms, cudaStream_t stream) {
    const int rows = a8_row_count(max_q_len * (long long)(a.num_heads / a.num_kv_heads));
    return rows == 4   ? a8_rows<T, 4, PARTS>(a, tokens, max_q_len, depth, n_sms, stream)
           : rows == 8 ? a8_rows<T, 8, PARTS>(a, tokens, max_q_len, depth, n_sms, stream)
                       : a8_rows<T, A8_HD <= 128 ? 16 : 8, PARTS>(a, tokens, max_q_len, depth, n_sms, stream);
}
template <typename T, int PARTS>
static int a8_singles(const A8Args& a, int max_ctx_len, int n_sms, int form, cudaStream_t stream) {
    const int G = a.num_heads / a.num_kv_heads, rows = a8_row_count(G);
    if (a8_few((long long)a.n_reqs * a.num_kv_heads * ((G + rows - 1) / rows), a8_tiles(max_ctx_len, a.window, 1), n_sms, form))
        return a8_portions<T, PARTS>(a, a.n_reqs, 1, max_ctx_len, n_sms, stream);
    return rows == 4 ? a8_stream<T, 4, PARTS>(a, n_sms, stream) : rows == 8 ? a8_stream<T, 8, PARTS>(a, n_sms, stream)
                                                                            : a8_stream<T, A8_HD <= 128 ? 16 : 8, PARTS>(a, n_sms, stream);
}

// Requests [0, n_decode) bring one token each, [n_decode, n_reqs) up to max_q_len; `portions`: about how many tokens the latter bring
// and, times 2^32, how deep they are; 0: the former only.
// Arguments packed, 8 bytes each, as the calls of cache_8bit.cu.
struct A8Call {
    const void *q, *k_cache, *v_cache;
    const float *k_scale, *v_scale;
    const int *block_table, *q_start, *ctx_lens;
    void *out, *scratch;
    const float* sinks;
    void* stream;
    long long dtype, q_stride, pages, max_blocks, scratch_bytes, n_decode, n_reqs, portions, max_q_len, max_ctx_len, num_heads,
        num_kv_heads, page_size, window, n_sms, form;
    double scale;
};
extern "C" int A8_SYM(rv_paged_attention_8bit)(const A8Call* c) {
    const void *q = c->q, *k_cache = c->k_cache, *v_cache = c->v_cache;
    void *out = c->out, *scratch = c->scratch, *stream = c->stream;
    const float *k_scale = c->k_scale, *v_scale = c->v_scale, *sinks = c->sinks, scale = (float)c->scale;
    const int *block_table = c->block_table, *q_start = c->q_start, *ctx_lens = c->ctx_lens;
    const long long q_stride = c->q_stride, pages = c->pages, scratch_bytes = c->scratch_bytes;
    for (const long long v : {c->max_blocks, c->n_reqs, c->max_q_len, c->max_ctx_len, c->num_heads, c->page_size, c->window})
        if (v > 0x7fffffff) A8_FAIL("paged_attention_8bit: bad sizes");
    const int dtype = (int)c->dtype, max_blocks = (int)c->max_blocks, n_decode = (int)c->n_decode, n_reqs = (int)c->n_reqs;
    const long long portions = c->portions & 0xffffffff;
    const int depth = (int)(c->portions >> 32);
    const int max_q_len = (int)c->max_q_len, max_ctx_len = (int)c->max_ctx_len;
    const int num_heads = (int)c->num_heads, num_kv_heads = (int)c->num_kv_heads, page_size = (int)c->page_size;
    const int window = (int)c->window, n_sms = (int)c->n_sms, form = (int)c->form;
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads)
        A8_FAIL("paged_attention_8bit: invalid head counts: %d query, %d KV", num_heads, num_kv_heads);
    if (n_decode < 0 || n_reqs < n_decode || max_q_len < 0 || max_ctx_len < 0 || max_blocks < 0 || page_size <= 0 || window < 0 ||
        n_sms <= 0 || pages < 0)
        A8_FAIL("paged_attention_8bit: bad sizes");
    if (n_reqs > 65535 || num_kv_heads > 65535) A8_FAIL("paged_attention_8bit: too many requests or heads");
    if (pages * num_kv_heads * page_size >= 0xffffffffll) A8_FAIL("paged_attention_8bit: more rows than 32 bits count");
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) % 16) A8_FAIL("paged_attention_8bit: pages must be 16-byte aligned");
    if (A8_SYM(rv_paged_attention_8bit_scratch_bytes)(n_decode, max_ctx_len, num_heads, num_kv_heads, window, n_sms, form) > scratch_bytes)
        A8_FAIL("paged_attention_8bit: scratch too small");
    A8Args a = {q, (const signed char*)k_cache, (const signed char*)v_cache, k_scale, v_scale, block_table, q_start, ctx_lens, sinks,
                out, (float*)scratch, nullptr, q_stride, pages, max_blocks, 0, n_decode, num_heads, num_kv_heads, page_size,
                (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1, window, 0, 0, scale * 1.4426950408889634f};
    a.vec = (uintptr_t)q % 16 == 0 && q_stride * (dtype == RV_DTYPE_F32 ? 4 : 2) % 16 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype != RV_DTYPE_F32 && dtype != RV_DTYPE_BF16) A8_FAIL("paged_attention_8bit: unknown dtype code %d", dtype);
    if (n_decode > 0) {
        const int rc = dtype == RV_DTYPE_BF16 ? a8_singles<__nv_bfloat16, 1>(a, max_ctx_len, n_sms, form, s)
                                              : a8_singles<float, 2>(a, max_ctx_len, n_sms, form, s);
        if (rc) return rc;
    }
    if (portions > 0 && n_reqs > n_decode && max_q_len > 0) {
        a.first_req = n_decode;
        a.n_reqs = n_reqs - n_decode;
        const int rc = dtype == RV_DTYPE_BF16 ? a8_portions<__nv_bfloat16, 1>(a, portions, max_q_len, depth, n_sms, s)
                                              : a8_portions<float, 2>(a, portions, max_q_len, depth, n_sms, s);
        if (rc) return rc;
    }
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) A8_FAIL("paged_attention_8bit: %s", cudaGetErrorString(e));
    return 0;
}
