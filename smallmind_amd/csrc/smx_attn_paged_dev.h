// smx_attn_paged_dev.h -- what the attention over the paged KV cache (k_attn_paged.hip) and the sum of the weights that
// positions receive (k_attn_mass.hip) share: a batch's rows and what they see, matrix operands, scores.  Compiled once per
// row width and element type of the cache.
#pragma once

#include <type_traits>

#include "smx_attn_paged.h"
#include "smx_device.h"
#include "smx_internal.h"

#if !defined(SMX_PG_W) || !defined(SMX_PG_BF16)
#error "SMX_PG_W: the cache's row width, SMX_PG_BF16: its type"
#endif

namespace smx {

namespace {

constexpr int W = SMX_PG_W;
constexpr bool BF16 = SMX_PG_BF16;
constexpr int NK = W / 16;               // matrix instructions along a K row
constexpr int ND = W / 32;               // 32-dim groups of the output
constexpr int ROW = 2 * W;               // bytes
constexpr float kNegInf = -__builtin_huge_valf();
typedef std::conditional_t<BF16, __bf16, _Float16> elem;
typedef elem elem2 __attribute__((ext_vector_type(2)));
typedef elem elem4 __attribute__((ext_vector_type(4)));
typedef elem elem8 __attribute__((ext_vector_type(8)));
typedef float float16v __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float16v mfma(elem8 a, elem8 b, float16v c)
{
    if constexpr (BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ float max_halves(float v)   // over the two lanes of a row
{
    const float2 p = swap32(v, v);
    return fmaxf(p.x, p.y);
}
__device__ __forceinline__ float sum_halves(float v)
{
    const float2 p = swap32(v, v);
    return p.x + p.y;
}

__device__ __forceinline__ int by_group(int id, double inv_group) { return (int)(((double)id + 0.5) * inv_group); }

// 16 bytes per lane from g to LDS at l + 16 * lane
__device__ __forceinline__ void to_lds(const void *g, void *l)
{
    const uint32_t la = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)l;
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "{m0}"(la) : "memory");
}
// The wave's loads have landed, its LDS reads are done.
__device__ __forceinline__ void wait_all()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(7 << 4);
    asm volatile("" ::: "memory");
}

// ---- a batch's sequences ---------------------------------------------------------------------------
struct Seq {
    int start, rows;       // first token; rows per KV head of the tokens taken
    int first, len;        // position of the first new token, positions in all
    int pre;               // positions that every token sees
    const int32_t *table;
};

__device__ __forceinline__ Seq seq_of(const AttnPgArgs &a, int b)
{
    Seq s;
    s.start = min(max(ld_uniform(a.starts + b), 0), a.n_tok);
    const int end = min(max(ld_uniform(a.starts + b + 1), s.start), a.n_tok);
    s.rows = min(end - s.start, a.max_q) * a.group;
    s.len = min(max(ld_uniform(a.lens + b), 0), a.max_len);
    s.first = s.len - (end - s.start);
    s.pre = a.prefix ? min(max(ld_uniform(a.prefix + b), 0), s.len) : 0;
    s.table = a.tables + (int64_t)b * a.table_stride;
    return s;
}

// What the rows of tokens at positions t0 .. t1 go through: tiles [0, pre) and [from, end), `count` in all.
struct Range {
    int pre, from, end, count;
    __device__ __forceinline__ int tile(int i) const { return i < pre ? i : i - pre + from; }
};
__device__ __forceinline__ Range range_of(const AttnPgArgs &a, const Seq &s, int t0, int t1)
{
    Range r;
    const int lo = a.window > 0 ? max(0, t0 - a.window + 1) : 0, hi = min(max(t1 + 1, 0), s.len);
    r.pre = (s.pre + kPgTile - 1) / kPgTile;
    r.from = max(lo / kPgTile, r.pre);
    r.end = max((hi + kPgTile - 1) / kPgTile, r.from);
    r.count = r.pre + r.end - r.from;
    return r;
}

// A lane's row: what it sees are positions below pre, and those from lo to below hi.
struct Row {
    int token, head;
    int t, lo, hi;
    bool valid;
};
__device__ __forceinline__ Row row_of(const AttnPgArgs &a, const Seq &s, int kv_head, int id)
{
    Row r;
    r.valid = id < s.rows;
    const int i = max(min(id, s.rows - 1), 0), tok = by_group(i, a.inv_group);
    r.token = s.start + tok;
    r.head = kv_head * a.group + i - tok * a.group;
    r.t = s.first + tok;
    r.lo = a.window > 0 ? max(0, r.t - a.window + 1) : 0;
    r.hi = min(max(r.t + 1, 0), s.len);
    return r;
}

// Rows of 16 positions, block `blk` of a sequence, in KV head h: the address, and whether the cache has the page.
struct Rows16 {
    const uint8_t *p;
    bool there;
};
__device__ __forceinline__ Rows16 rows16(const AttnPgArgs &a, const Seq &s, int head, int blk)
{
    // (beyond the last position: its block again, which no table lacks)
    const int j = max(min(blk, (s.len + kPgGroup - 1) / kPgGroup - 1), 0) * kPgGroup;
    const int pg = ld_uniform(s.table + (j >> a.page_shift));
    Rows16 r;
    r.there = (unsigned)pg < (unsigned)a.c.n_pages;
    r.p = a.c.k_row(r.there ? pg : 0, head, j & (a.c.page - 1));
    return r;
}

// ---- operands --------------------------------------------------------------------------------------
// Parts of a row of queries and of weights: 16-bit queries one, fp32 ones two of fp16 or three of bf16.
template <bool F32> constexpr int kParts = F32 ? (BF16 ? 3 : 2) : 1;

template <int NP>
__device__ __forceinline__ void split(float f, elem (&p)[NP])
{
    p[0] = (elem)f;
    if constexpr (NP > 1) {
        const float r = f - (float)p[0];
        p[1] = (elem)r;
        if constexpr (NP > 2) p[2] = (elem)(r - (float)p[1]);
    }
}

template <bool F32> struct Query {
    elem8 q[kParts<F32>][NK];
    float unit;            // of the products
};

template <bool F32>
__device__ __forceinline__ void load_q(const AttnPgArgs &a, const Row &r, int h, Query<F32> &Q)
{
    const int64_t at = (int64_t)r.token * a.q_stride + (int64_t)r.head * a.c.hd;
    Q.unit = 1.0f;
    if constexpr (!F32) {
        uint32_t top = 0;
#pragma unroll
        for (int n = 0; n < NK; n++) {
            const int d = 16 * n + 8 * h;
            uint16_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (d < a.c.hd) {
                const uint16_t *p = (const uint16_t *)a.q + at + d;
                if (a.q_vec) {
                    __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 16);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = p[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, (uint32_t)(v[e] & 0x7FFF));
            __builtin_memcpy(&Q.q[0][n], v, 16);
        }
        // a row that holds a NaN or an infinity is NaN
        const bool bad = max_halves(top >= (BF16 ? 0x7F80u : 0x7C00u) ? 1.0f : 0.0f) > 0.0f;
        if (bad) Q.unit = __builtin_nanf("");
    } else {
        float f[NK][8];
        uint32_t top = 0;
#pragma unroll
        for (int n = 0; n < NK; n++) {
            const int d = 16 * n + 8 * h;
#pragma unroll
            for (int e = 0; e < 8; e++) f[n][e] = 0.0f;
            if (d < a.c.hd) {
                const float *p = (const float *)a.q + at + d;
                if (a.q_vec) {
                    __builtin_memcpy(f[n], __builtin_assume_aligned(p, 16), 32);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) f[n][e] = p[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(f[n][e]) & 0x7FFFFFFFu);
        }
        const bool bad = max_halves(top > 0x7F7FFFFFu ? 1.0f : 0.0f) > 0.0f;
        float mul = 1.0f;
        if constexpr (!BF16) {
            // the power of two that brings the row's largest below 2^15
            const float amax = fmaxf(max_halves(__uint_as_float(min(top, 0x7F7FFFFFu))), 7.8886090522101181e-31f);
            const uint32_t e = __float_as_uint(amax) & 0x7F800000u;
            mul = __uint_as_float((268u << 23) - e);
            Q.unit = __uint_as_float(e) * (1.0f / 16384.0f);
        }
        if (bad) Q.unit = __builtin_nanf("");
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                elem p[kParts<F32>];
                split(f[n][e] * mul, p);
#pragma unroll
                for (int k = 0; k < kParts<F32>; k++) Q.q[k][n][e] = p[k];
            }
    }
}

// Where a lane finds its operands among rows in LDS.  K: row r = lane % 32 of 32, unit 2 n + h.  V^T: for dims
// 32 d + lane % 32 the positions 4 h + .. and 8 + 4 h + .. of 16, each from an 8-byte piece that sixteen lanes transpose
// between them.
constexpr int KO = W % 64 == 0 ? 4 : 2;   // places after which pg_unit's turn of the units repeats
struct LaneAt {
    uint32_t k[KO], v[2][2];
    __device__ __forceinline__ LaneAt(int lane)
    {
        const int r = lane & 31, h = lane >> 5;
#pragma unroll
        for (int j = 0; j < KO; j++) k[j] = r * ROW + 16 * pg_unit(W, 2 * j + h, r);
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int key = 8 * p + 4 * h + ((lane & 15) >> 2), u = 4 * j + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
                v[p][j] = key * ROW + 16 * pg_unit(W, u, key) + 8 * (lane & 1);
            }
    }
    // of the 32 rows at `rows`, operand n
    __device__ __forceinline__ elem8 key(const uint8_t *rows, int n) const
    {
        return *(const elem8 *)(rows + k[n % KO] + 32 * KO * (n / KO));
    }
    // of the 16 rows at `rows`, dims 32 d ..
    __device__ __forceinline__ elem8 val(const uint8_t *rows, int d) const
    {
        typedef short4v __attribute__((address_space(3))) *at;
        union { short4v s[2]; elem8 e; } r;
#pragma unroll
        for (int p = 0; p < 2; p++)
            r.s[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(rows + v[p][d % 2] + 128 * (d / 2)));
        return r.e;
    }
};
static_assert(W % 64 == 0 || W == 32 || W == 96, "pg_unit turns whole sets of units");

// ---- scores ----------------------------------------------------------------------------------------
// tanh: its series below 0.4 (the next term is less than 2^-24 of the value there), else by an exponential.
__device__ __forceinline__ float tanh_of(float y)
{
    const float t = fabsf(y), z = y * y;
    float p = -1382.0f / 155925.0f;
    p = __builtin_fmaf(p, z, 62.0f / 2835.0f);
    p = __builtin_fmaf(p, z, -17.0f / 315.0f);
    p = __builtin_fmaf(p, z, 2.0f / 15.0f);
    p = __builtin_fmaf(p, z, -1.0f / 3.0f);
    const float small = __builtin_fmaf(p * z, t, t);
    const float e = __builtin_amdgcn_exp2f(t * -2.8853900817779268f);
    const float large = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
    return copysignf(t < 0.4f ? small : large, y);
}

// How a lane's products become exponents of 2: x * c, or with a cap or slopes x itself after shape().
struct Shape {
    float c;             // what is left to multiply by
    float in;            // products to scores (shaped)
    float slope;
    bool shaped;
    __device__ __forceinline__ Shape(const AttnPgArgs &a, const Row &r, float unit)
    {
        shaped = a.cap_in != 0.0f || a.slopes;
        in = (a.cap_in != 0.0f ? a.cap_in : a.scale_log2e) * unit;
        c = shaped ? 1.0f : in;
        slope = a.slopes ? a.slopes[r.head] * 1.4426950408889634f : 0.0f;
    }
};

// Position (of 32) of a lane's element i.
__device__ __forceinline__ int pos32(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// x of 32 positions from `at` on.
__device__ __forceinline__ void shape(const AttnPgArgs &a, const Shape &S, float16v &x, const Row &r, int at, int h)
{
    if (a.cap_in != 0.0f) {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = tanh_of(x[i] * S.in) * a.cap_out;
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] *= S.in;
    }
    if (a.slopes) {
        const int away = r.t - at - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __builtin_fmaf(-S.slope, fabsf((float)(away - pos32(i, 0))), x[i]);
    }
}

// -inf where the row does not see: there[b]: the cache has the page of positions 16 b ..
__device__ __forceinline__ void mask(float16v &x, const Row &r, int pre, int at, int h, bool there0, bool there1)
{
    const int p0 = at + 4 * h;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int p = p0 + pos32(i, 0);
        const bool see = (p < pre || (p >= r.lo && p < r.hi)) && (i < 8 ? there0 : there1);
        x[i] = see ? x[i] : kNegInf;
    }
}

// Whether every row of a wave sees all of positions [at, at + n), or none.  lo and hi of the wave's rows: the lowest
// and the highest.
struct Bounds {
    int lo0, lo1, hi0, hi1;
    __device__ __forceinline__ bool whole(int pre, int at, int n) const { return at + n <= pre || (at >= lo1 && at + n <= hi0); }
    __device__ __forceinline__ bool none(int pre, int at, int n) const { return at >= pre && (at >= hi1 || at + n <= lo0); }
};
__device__ __forceinline__ Bounds bounds_of(const AttnPgArgs &a, const Seq &s, int row0, int n)
{
    // (a later token's bounds are no lower)
    const Row first = row_of(a, s, 0, row0), last = row_of(a, s, 0, row0 + n - 1);
    Bounds b;
    b.lo0 = __builtin_amdgcn_readfirstlane(first.lo), b.lo1 = __builtin_amdgcn_readfirstlane(last.lo);
    b.hi0 = __builtin_amdgcn_readfirstlane(first.hi), b.hi1 = __builtin_amdgcn_readfirstlane(last.hi);
    return b;
}

}  // namespace

}  // namespace smx
