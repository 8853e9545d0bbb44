// k_paged_write.hip -- rows into the paged KV cache (smx_paged.h) and back: norms of queries and keys for each head, the
// rotation by position and the write in one pass; without a cache the same from rows to rows.
//
// Mathematics.  x' = x / sqrt(mean x^2 + eps) * gamma per head, then each pair (a, b) of channels becomes
// (a cos - b sin, a sin + b cos) with the angle of the pair's axis, all in fp32, rounded once.  V is rounded and kept.
//
// Layout.  A lane holds 8 channels of a row; a row's lanes (a power of two of them) sum its squares by lane exchanges.  Where
// pairs lie half a row apart, a lane reads its partners' channels itself (from the L1 they have just come to), which leaves
// head_dim and the rotated width free of any rule on lanes.  A work item is one query row, or one K row with its V row:
// whether V is finite decides what K holds.
#include "smx_device.h"
#include "smx_internal.h"

namespace smx {

namespace {

template <int TYPE> struct Elem { typedef float type; };
template <> struct Elem<PG_F16> { typedef _Float16 type; };
template <> struct Elem<PG_BF16> { typedef __bf16 type; };

// Eight consecutive values from element `at` on.
template <int TYPE>
__device__ __forceinline__ void load8(float (&x)[8], const void *p, int64_t at, bool vec)
{
    typedef typename Elem<TYPE>::type E;
    const E *e = (const E *)p + at;
    if (vec) {
        typedef E E8 __attribute__((ext_vector_type(8)));
        E8 v;
        __builtin_memcpy(&v, __builtin_assume_aligned(e, 16), sizeof(v));
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = (float)e[i];
    }
}

template <typename E>
__device__ __forceinline__ void store8_as(void *p, int64_t at, const float (&x)[8], bool vec)
{
    E *e = (E *)p + at;
    if (vec) {
        typedef E E8 __attribute__((ext_vector_type(8)));
        E8 v;
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = (E)x[i];
        __builtin_memcpy(__builtin_assume_aligned(e, 16), &v, sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = (E)x[i];
    }
}

__device__ __forceinline__ void store8(int type, void *p, int64_t at, const float (&x)[8], bool vec)
{
    if (type == PG_F32) store8_as<float>(p, at, x, vec);
    else if (type == PG_F16) store8_as<_Float16>(p, at, x, vec);
    else store8_as<__bf16>(p, at, x, vec);
}

// x rounded to the cache's type; bad: one of them is not finite.
struct Unit {
    uint4 u;
    bool bad;
};
__device__ __forceinline__ Unit rounded(int bf16, const float (&x)[8])
{
    uint16_t h[8];
    bool bad = false;
    const uint32_t top = bf16 ? 0x7F80u : 0x7C00u;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        h[i] = bf16 ? __builtin_bit_cast(uint16_t, (__bf16)x[i]) : __builtin_bit_cast(uint16_t, (_Float16)x[i]);
        bad |= (h[i] & top) == top;
    }
    Unit r;
    r.bad = bad;
    __builtin_memcpy(&r.u, h, 16);
    return r;
}

// Cosines and sines of the pairs of this lane's channels: N of them from pair j0 on.
template <int N>
__device__ __forceinline__ void angles(const PgRotation &r, int n_tok, int t, int j0, float (&c)[N], float (&s)[N])
{
    int a0 = 0;
    while (a0 < 3 && j0 >= r.ends[a0]) a0++;
    if (j0 + N <= r.ends[a0] && r.vec && (j0 & 3) == 0) {
        const int p = r.pos[(int64_t)a0 * n_tok + t];
        const bool in = (unsigned)p < (unsigned)r.n_pos;
        const int64_t at = in ? (int64_t)p * r.half + j0 : 0;   // (a position outside: the first row, not used)
        const float bad = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 cv = *(const float4 *)(r.cos + (in ? at + i : 0)), sv = *(const float4 *)(r.sin + (in ? at + i : 0));
            c[i] = in ? cv.x : bad, c[i + 1] = in ? cv.y : bad, c[i + 2] = in ? cv.z : bad, c[i + 3] = in ? cv.w : bad;
            s[i] = in ? sv.x : bad, s[i + 1] = in ? sv.y : bad, s[i + 2] = in ? sv.z : bad, s[i + 3] = in ? sv.w : bad;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const int j = min(j0 + i, r.half - 1);   // (channels beyond the rotated ones: not used)
        int a = a0;
        while (a < 3 && j >= r.ends[a]) a++;
        const int p = r.pos[(int64_t)a * n_tok + t];
        const bool in = (unsigned)p < (unsigned)r.n_pos;
        const int64_t at = in ? (int64_t)p * r.half + j : 0;
        c[i] = in ? r.cos[at] : __builtin_nanf("");
        s[i] = in ? r.sin[at] : __builtin_nanf("");
    }
}

// This lane's channels d0 .. d0 + 7 of the row at `at` of p, normed and turned.  `on`: the lane has channels.
template <int TYPE>
__device__ __forceinline__ void turned(const PgWriteArgs &a, float (&y)[8], const void *p, int64_t at, int d0, int t,
                                       const float *gamma, bool on)
{
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) load8<TYPE>(x, p, at + d0, a.vec);
    float r = 1.0f;
    if (gamma) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) sq = __builtin_fmaf(x[i], x[i], sq);
        for (int o = (1 << a.group_shift) >> 1; o > 0; o >>= 1) sq += __shfl_xor(sq, o, 64);
        r = 1.0f / sqrtf(sq / (float)a.hd + a.eps);
    }
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = gamma && on ? x[i] * r * gamma[d0 + i] : x[i];
    const int half = a.rot.half;
    if (!on || d0 >= 2 * half) return;
    if (!a.rot.halves) {
        float c[4], s[4];
        angles<4>(a.rot, a.n_tok, t, d0 >> 1, c, s);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if (d0 + i >= 2 * half) break;
            const float u = y[i], v = y[i + 1];
            y[i] = u * c[i >> 1] - v * s[i >> 1];
            y[i + 1] = u * s[i >> 1] + v * c[i >> 1];
        }
        return;
    }
    if ((half & 7) == 0) {   // the eight partners lie together
        const bool low = d0 < half;
        const int e0 = low ? d0 + half : d0 - half;
        float z[8], c[8], s[8];
        load8<TYPE>(z, p, at + e0, a.vec);
        angles<8>(a.rot, a.n_tok, t, low ? d0 : e0, c, s);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = gamma ? z[i] * r * gamma[e0 + i] : z[i];
            y[i] = low ? y[i] * c[i] - w * s[i] : w * s[i] + y[i] * c[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int d = d0 + i;
        if (d >= 2 * half) break;
        const bool low = d < half;
        const int e = low ? d + half : d - half;
        float c[1], s[1];
        angles<1>(a.rot, a.n_tok, t, low ? d : e, c, s);
        const float z = (float)((const typename Elem<TYPE>::type *)p)[at + e];
        const float w = gamma ? z * r * gamma[e] : z;
        y[i] = low ? y[i] * c[0] - w * s[0] : w * s[0] + y[i] * c[0];
    }
}

// An item is 1 << group_shift lanes; a.groups items per token: the query heads, then the KV heads.
template <int TYPE>
__global__ __launch_bounds__(256) void k_paged_write(const PgWriteArgs a)
{
    const int lane = threadIdx.x & ((1 << a.group_shift) - 1);
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> a.group_shift;
    const int64_t tt = item / a.groups;
    if (tt >= a.n_tok) return;           // (whole items: the lanes that exchange stay together)
    const int t = (int)tt, g = (int)(item - tt * a.groups), d0 = lane * 8;
    const bool on = d0 < a.hd;
    const int nq = a.q ? a.n_head : 0;
    float y[8];
    if (g < nq) {
        turned<TYPE>(a, y, a.q, t * a.q_stride + (int64_t)g * a.hd, d0, t, a.q_gamma, on);
        if (on) store8(a.out_type, a.q_out, ((int64_t)t * a.n_head + g) * a.hd + d0, y, a.vec);
        return;
    }
    const int head = g - nq;
    if (!a.c.base) {
        turned<TYPE>(a, y, a.k, t * a.k_stride + (int64_t)head * a.hd, d0, t, a.k_gamma, on);
        if (on) store8(a.out_type, a.k_out, ((int64_t)t * a.n_kv + head) * a.hd + d0, y, a.vec);
        return;
    }
    const int place = a.places[t];
    if (place < 0 || place >= a.c.n_pages * a.c.page) return;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) load8<TYPE>(v, a.v, t * a.v_stride + (int64_t)head * a.hd + d0, a.vec);
    turned<TYPE>(a, y, a.k, t * a.k_stride + (int64_t)head * a.hd, d0, t, a.k_gamma, on);
    Unit ku = rounded(a.c.bf16, y), vu = rounded(a.c.bf16, v);
    int bad = on && (ku.bad || vu.bad);
    for (int o = (1 << a.group_shift) >> 1; o > 0; o >>= 1) bad |= __shfl_xor(bad, o, 64);
    if (!on) return;
    if (bad) {
        ku.u = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
        vu.u = make_uint4(0, 0, 0, 0);
    }
    const int r = place & (a.c.page - 1);
    uint8_t *row = a.c.k_row(place / a.c.page, head, r) + 16 * pg_unit(a.c.w, lane, r);
    *(uint4 *)row = ku.u;
    *(uint4 *)(row + a.c.v_off()) = vu.u;
}

// Reads rows back: [n_tok][n_kv][hd] in the cache's type; zeros for places that it does not have, NaN for a position
// that was not finite.
__global__ __launch_bounds__(256) void k_paged_read(const PgView c, const int32_t *places, int n_tok, uint16_t *k, uint16_t *v)
{
    const int per = c.hd / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row_id = i / per;
    const int u = (int)(i - row_id * per);
    const int64_t t = row_id / c.n_kv;
    if (t >= n_tok) return;
    const int head = (int)(row_id - t * c.n_kv), place = places[t];
    uint4 ku = make_uint4(0, 0, 0, 0), vu = ku;
    if (place >= 0 && place < c.n_pages * c.page) {
        const int r = place & (c.page - 1);
        const uint8_t *row = c.k_row(place / c.page, head, r) + 16 * pg_unit(c.w, u, r);
        ku = *(const uint4 *)row;
        vu = *(const uint4 *)(row + c.v_off());
        if ((ku.x & 0x7FFFu) == 0x7FFFu) vu = ku;
    }
    ((uint4 *)k)[i] = ku;
    ((uint4 *)v)[i] = vu;
}

}  // namespace

hipError_t launch_paged_write(PgWriteArgs a, int in_type, hipStream_t s)
{
    a.group_shift = 0;
    while ((8 << a.group_shift) < a.hd) a.group_shift++;
    a.groups = (a.q ? a.n_head : 0) + (a.k ? a.n_kv : 0);
    const unsigned blocks = (unsigned)((((int64_t)a.n_tok * a.groups << a.group_shift) + 255) / 256);
    if (in_type == PG_F32) k_paged_write<PG_F32><<<blocks, 256, 0, s>>>(a);
    else if (in_type == PG_F16) k_paged_write<PG_F16><<<blocks, 256, 0, s>>>(a);
    else k_paged_write<PG_BF16><<<blocks, 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_paged_read(const PgView &c, const int32_t *places, int n_tok, void *k, void *v, hipStream_t s)
{
    const int64_t n = (int64_t)n_tok * c.n_kv * (c.hd / 8);
    k_paged_read<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(c, places, n_tok, (uint16_t *)k, (uint16_t *)v);
    return hipGetLastError();
}

}  // namespace smx
