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

// 16 bytes per lane from g + off (g the same in every lane) to LDS at l + 16 * lane
__device__ __forceinline__ void to_lds(const uint8_t *g, uint32_t off, void *l)
{
    const uint32_t la = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void *)l;
    asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(g), "{m0}"(la) : "memory");
}
// All but the wave's last N loads have landed, its LDS reads are done.
template <int N>
__device__ __forceinline__ void wait_loads()
{
    static_assert(N >= 0 && N < 64, "vmcnt has 6 bits");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));
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

// The sequence that is n-th by length, the longest first, among the 64 that n is one of.
__device__ __forceinline__ int nth_longest(const AttnPgArgs &a, int n)
{
    const int lane = threadIdx.x & 63, b0 = n & ~63, count = min(64, a.n_seq - b0);
    const int len = lane < count ? a.lens[b0 + lane] : 0;
    int rank = lane < count ? 0 : 64;
    for (int j = 0; j < count; j++) {
        const int l = __builtin_amdgcn_readlane(len, j);
        rank += l > len || (l == len && j < lane);
    }
    return b0 + __builtin_ctzll(__ballot(rank == n - b0));
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

// A lane's row: a token at position t.  What it sees are positions below the sequence's
// pre, and those from lo_of to below hi_of.
struct Row {
    int token, head, t;
    bool valid;
};
__device__ __forceinline__ int lo_of(const AttnPgArgs &a, int t) { return a.window > 0 ? max(0, t - a.window + 1) : 0; }
__device__ __forceinline__ int hi_of(const Seq &s, int t) { return min(max(t + 1, 0), s.len); }
__device__ __forceinline__ Row row_of(const AttnPgArgs &a, const Seq &s, int kv_head, int id)
{
    Row r;
    r.valid = id < s.rows;
    const int i = max(min(id, s.rows - 1), 0), tok = by_group(i, a.inv_group);
    r.token = s.start + tok;
    r.head = kv_head * a.group + i - tok * a.group;
    r.t = s.first + tok;
    return r;
}

// Rows of 16 positions of a sequence in one KV head: the address, and whether the cache has the page.
struct Rows16 {
    const uint8_t *p;
    bool there;
};

// A wave's view of a sequence's page table: lane l has the page of the 16 positions 64 * win + l, and of those 64 further on, so
// that a tile's pages are at hand when its rows are asked for.
struct Pages {
    int win, id, next;
    uint64_t ok;           // which of them the cache has
    int last;              // (beyond the last position: its page again, which no table lacks)
    const uint8_t *base;   // of the KV head in page 0
    uint32_t kb;           // from page to page

    __device__ __forceinline__ int at(const AttnPgArgs &a, const Seq &s, int w) const
    {
        return s.table[(max(min(64 * w + (int)(threadIdx.x & 63), last), 0) * kPgGroup) >> a.page_shift];
    }
    __device__ __forceinline__ void check(const AttnPgArgs &a) { ok = __ballot((unsigned)id < (unsigned)a.c.n_pages); }
    __device__ __forceinline__ Pages(const AttnPgArgs &a, const Seq &s, int head, int blk)
    {
        base = a.c.base + head * a.c.head_bytes();
        kb = (uint32_t)(a.c.n_kv * (a.c.head_bytes() >> 10));
        last = (s.len + kPgGroup - 1) / kPgGroup - 1;
        win = blk >> 6;
        id = at(a, s, win), next = at(a, s, win + 1);
        check(a);
    }
    // block blk's window
    __device__ __forceinline__ void go(const AttnPgArgs &a, const Seq &s, int blk)
    {
        const int w = blk >> 6;
        if (w == win) return;
        id = w == win + 1 ? next : at(a, s, w);
        next = at(a, s, w + 1);
        win = w;
        check(a);
    }
    __device__ __forceinline__ Rows16 rows(const AttnPgArgs &a, int blk) const
    {
        Rows16 r;
        r.there = ok >> (blk & 63) & 1;
        const uint32_t pg = r.there ? __builtin_amdgcn_readlane(id, blk & 63) : 0;
        r.p = base + (((uint64_t)pg * kb << 10) + (uint32_t)(((min(blk, last) * kPgGroup) & (a.c.page - 1)) * ROW));
        return r;
    }
};

// ---- operands --------------------------------------------------------------------------------------
// Parts of a row of queries and of weights: 16-bit queries one, fp32 ones two of fp16 or three of bf16.
template <bool F32> constexpr int kParts = F32 ? (BF16 ? 3 : 2) : 1;

// Two values' parts, each the nearest to what the ones before leave.
template <int NP>
__device__ __forceinline__ void split(float f, float g, elem2 (&p)[NP])
{
    p[0] = elem2{(elem)f, (elem)g};
    if constexpr (NP == 2) {
        // what is left, exactly, the half read as fp16 by the same instruction (written as such, the compiler converts it first)
        float a, b;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(a) : "v"(p[0]), "v"(f));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(b) : "v"(p[0]), "v"(g));
        p[1] = elem2{(elem)a, (elem)b};
    } else if constexpr (NP == 3) {
        float a = f - (float)p[0][0], b = g - (float)p[0][1];
        p[1] = elem2{(elem)a, (elem)b};
        p[2] = elem2{(elem)(a - (float)p[1][0]), (elem)(b - (float)p[1][1])};
    }
}
static_assert(BF16 || kParts<true> == 2, "two parts are fp16");

template <bool F32> struct Query {
    elem8 q[kParts<F32>][NK];
    float unit;            // of the products
};

// A row that gives NaN: its products become that, and only they, so that what the row does not see is masked as ever, and a row that sees
// nothing stays one.  (One element is enough: NaN times 0 is NaN.)
template <bool F32>
__device__ __forceinline__ void spoil(Query<F32> &Q, bool bad)
{
    Q.q[0][0][0] = bad ? (elem)__builtin_nanf("") : Q.q[0][0][0];
}

// CHECK: a row that holds a NaN or an infinity is spoilt.
template <bool F32, bool CHECK = true>
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
            __builtin_memcpy(&Q.q[0][n], v, 16);
            if constexpr (CHECK) {
#pragma unroll
                for (int e = 0; e < 8; e++) top = max(top, (uint32_t)(v[e] & 0x7FFF));
            }
        }
        if constexpr (CHECK) spoil(Q, max_halves(top >= (BF16 ? 0x7F80u : 0x7C00u) ? 1.0f : 0.0f) > 0.0f);
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
            const float amax = fmaxf(max_halves(__uint_as_float(min(top, 0x7F7FFFFFu))), a.q_least);
            const uint32_t e = __float_as_uint(amax) & 0x7F800000u;
            mul = __uint_as_float((268u << 23) - e);
            Q.unit = __uint_as_float(e) * (1.0f / 16384.0f);
        }
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                elem2 p[kParts<F32>];
                split(f[n][e] * mul, f[n][e + 1] * mul, p);
#pragma unroll
                for (int k = 0; k < kParts<F32>; k++) Q.q[k][n][e] = p[k][0], Q.q[k][n][e + 1] = p[k][1];
            }
        spoil(Q, bad);
    }
}

// Where a lane finds its operands among rows in LDS.  K: row r = lane % 32 of 32, unit 2 n + h.  V^T: for dims
// 32 d + lane % 32 the positions 4 h + .. and 8 + 4 h + .. of 16, each from an 8-byte piece that sixteen lanes transpose
// between them.  pg_unit's turn and a row's start leave the rest of a unit's number to be put in by one exclusive or.
struct LaneAt {
    uint32_t k0, v0;
    __device__ __forceinline__ LaneAt(int lane)
    {
        const int r = lane & 31, h = lane >> 5, key = 4 * h + ((lane & 15) >> 2), u = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        k0 = r * ROW + 16 * pg_unit(W, h, r);
        v0 = key * ROW + 16 * pg_unit(W, u, key) + 8 * (lane & 1);
    }
    // of the 32 rows at `rows`, operand n
    __device__ __forceinline__ elem8 key(const uint8_t *rows, int n) const
    {
        if constexpr (W % 64 == 0) return *(const elem8 *)(rows + (k0 ^ (32 * (n % 4))) + 128 * (n / 4));
        else return *(const elem8 *)(rows + (k0 ^ (32 * (n % 2))) + 64 * (n / 2));
    }
    // of the 16 rows at `rows`, dims 32 d ..
    __device__ __forceinline__ elem8 val(const uint8_t *rows, int d) const
    {
        typedef short4v __attribute__((address_space(3))) *at;
        union { short4v s[2]; elem8 e; } r;
#pragma unroll
        for (int p = 0; p < 2; p++) {
            // (eight rows further on the turn is the same, or unit 2's)
            const uint32_t o = W % 64 == 0 ? (v0 ^ (64 * (d % 2))) + 128 * (d / 2) : (v0 ^ (32 * p)) + 64 * d;
            r.s[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at)(rows + o + 8 * ROW * p));
        }
        return r.e;
    }
};
static_assert(W % 64 == 0 || W == 32 || W == 96, "pg_unit turns whole sets of units");

// ---- scores ----------------------------------------------------------------------------------------
// tanh: its series below 0.4 (the next term is 6.4e-8, some 2^-24, of the value there), else by an exponential.
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
    Shape() = default;
    __device__ __forceinline__ Shape(const AttnPgArgs &a, float slope_of, float unit)
    {
        shaped = a.cap_in != 0.0f || a.slopes;
        in = (a.cap_in != 0.0f ? a.cap_in : a.scale_log2e) * unit;
        c = shaped ? 1.0f : in;
        slope = slope_of * 1.4426950408889634f;
    }
};

// Position (of 32) of a lane's element i.
__device__ __forceinline__ int pos32(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// x of 32 positions from `at` on.  QUICK, for 16-bit outputs and caps up to kQuickCap: tanh is 1 - 2 / (1 + e^2y), off by up to 2^-21
// where the series keeps small values to 2^-24 of themselves: 2^-21 of the cap in a score, 2^-14 at most, which a weight's 8 or 11
// bits do not notice, for 5 instructions in place of 19.
constexpr float kQuickCap = 128.0f * 1.4426950408889634f;   // (as an exponent of 2)
template <bool QUICK>
__device__ __forceinline__ void shape(const AttnPgArgs &a, const Shape &S, float16v &x, int t, int at, int h)
{
    const float away = (float)(t - at - 4 * h);   // (exact: positions are below 2^24)
    if (QUICK && a.cap_in != 0.0f) {
        const float in = S.in * 2.8853900817779268f;
#pragma unroll
        for (int i = 0; i < 16; i++)
            x[i] = __builtin_fmaf(__builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x[i] * in)), -2.0f * a.cap_out, a.cap_out);
        if (a.slopes) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = __builtin_fmaf(-S.slope, fabsf(away - (float)pos32(i, 0)), x[i]);
        }
    } else if (!QUICK && a.cap_in != 0.0f) {
#pragma unroll
        for (int i = 0; i < 16; i++) {
            x[i] = tanh_of(x[i] * S.in) * a.cap_out;
            if ((i & 3) == 3) __builtin_amdgcn_sched_barrier(0);   // (four at a time: all at once take too many registers)
        }
        if (a.slopes) {
#pragma unroll
            for (int i = 0; i < 16; i++) x[i] = __builtin_fmaf(-S.slope, fabsf(away - (float)pos32(i, 0)), x[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __builtin_fmaf(x[i], S.in, -S.slope * fabsf(away - (float)pos32(i, 0)));
    }
}

// Of 32 positions from `at` on the row at t sees those whose bit is set, as a lane has them (its 16 in every second four).
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen(const AttnPgArgs &a, const Seq &s, int t, int at, int h, bool there0, bool there1)
{
    const uint32_t m = below(s.pre - at) | (below(hi_of(s, t) - at) & ~below(lo_of(a, t) - at));
    return (m & ((there0 ? 0xFFFFu : 0u) | (there1 ? 0xFFFF0000u : 0u))) >> (4 * h);
}
// -inf where it does not.
__device__ __forceinline__ void mask(float16v &x, uint32_t m)
{
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const uint32_t on = (uint32_t)__builtin_amdgcn_sbfe((int)m, pos32(i, 0), 1);   // all ones or none
        x[i] = __uint_as_float((__float_as_uint(x[i]) & on) | (0xFF800000u & ~on));
    }
}

// Whether every row of a wave sees all of positions [at, at + n), or none.  lo and hi of the wave's rows: the lowest
// and the highest.
struct Bounds {
    int lo0, lo1, hi0, hi1;
    __device__ __forceinline__ bool whole(int pre, int at, int n) const { return at + n <= pre || (at >= lo1 && at + n <= hi0); }
    __device__ __forceinline__ bool none(int pre, int at, int n) const { return at >= pre && (at >= hi1 || at + n <= lo0); }
};
__device__ __forceinline__ Bounds bounds_of(const AttnPgArgs &a, const Seq &s, int t0, int t1)   // the first row's t, the last one's
{
    t0 = __builtin_amdgcn_readfirstlane(t0), t1 = __builtin_amdgcn_readfirstlane(t1);
    return Bounds{lo_of(a, t0), lo_of(a, t1), hi_of(s, t0), hi_of(s, t1)};   // (a later token's are no lower)
}

}  // namespace

}  // namespace smx
