// k_paged_write.hip -- rows into the paged KV cache (smx_paged.h) and back: norms of queries and keys for each head, the
// rotation by position and the write in one pass; without a cache the same from rows to rows.
//
// Mathematics.  x' = x / sqrt(mean x^2 + eps) * gamma per head, then each pair (a, b) of channels becomes
// (a cos - b sin, a sin + b cos) with the angle of the pair's axis, all in fp32, rounded once.  V is rounded and kept.
//
// Layout.  A lane holds 8 channels of a row; a row's lanes (a power of two of them) sum its squares by lane exchanges.  A wave
// stays with one token, whose cosines and sines and the weights of the norms its lanes load once, and takes its rows in turn, the next
// ones on their way from memory.  Where pairs lie half a row apart, a lane reads its partners' channels itself (from the
// L1 they have just come to), which leaves head_dim and the rotated width free of any rule on lanes.  A work item is one
// query row, or one K row with its V row: whether V is finite decides what K holds.
#include <algorithm>

#include "smx_device.h"
#include "smx_internal.h"

namespace smx {

namespace {

template <int TYPE> struct Elem { typedef float type; };
template <> struct Elem<PG_F16> { typedef _Float16 type; };
template <> struct Elem<PG_BF16> { typedef __bf16 type; };

template <int TYPE> using Elem8 = typename Elem<TYPE>::type __attribute__((ext_vector_type(8)));

// Eight consecutive values from element `at` on, as they are.
template <int TYPE>
__device__ __forceinline__ Elem8<TYPE> load8(const void *p, int64_t at, bool vec)
{
    const typename Elem<TYPE>::type *e = (const typename Elem<TYPE>::type *)p + at;
    Elem8<TYPE> v;
    if (vec) {
        __builtin_memcpy(&v, __builtin_assume_aligned(e, 16), sizeof(v));
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = e[i];
    }
    return v;
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

// The sum over a row's lanes, 1 << shift of them (they run together, whatever the wave's other rows do).
__device__ __forceinline__ float row_sum(float v, int shift)
{
    if (shift > 0) v += dpp_mov<0xB1>(v);
    if (shift > 1) v += dpp_mov<0x4E>(v);
    if (shift > 2) v += dpp_mov<0x141>(v);
    if (shift > 3) v += dpp_mov<0x140>(v);
    if (shift > 4) v += swap16_other(v);
    return v;
}

// What a lane turns its channels with: y[i] c[i] + partner[i] s[i], the sign in s.
struct Turn {
    float c[8], s[8];
    int on;      // how many of the eight are turned
    int e0;      // first channel of the eight partners (halves, where these lie together)
};

__device__ __forceinline__ Turn turn_of(const PgWriteArgs &a, int d0)   // (the angles follow)
{
    Turn r;
    r.on = min(max(2 * a.rot.half - d0, 0), 8);
    r.e0 = d0 < a.rot.half ? d0 + a.rot.half : d0 - a.rot.half;
    return r;
}

__device__ __forceinline__ void angles_of(const PgWriteArgs &a, Turn &r, int t, int d0)
{
    const int half = a.rot.half;
    if (r.on == 0) return;
    if (!a.rot.halves) {
        float c[4], s[4];
        angles<4>(a.rot, a.n_tok, t, d0 >> 1, c, s);
#pragma unroll
        for (int i = 0; i < 8; i++) r.c[i] = c[i >> 1], r.s[i] = i & 1 ? s[i >> 1] : -s[i >> 1];
    } else if ((half & 7) == 0) {
        float s[8];
        angles<8>(a.rot, a.n_tok, t, min(d0, r.e0), r.c, s);
#pragma unroll
        for (int i = 0; i < 8; i++) r.s[i] = d0 < half ? -s[i] : s[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = d0 + i;
            float c[1], s[1];
            angles<1>(a.rot, a.n_tok, t, d < half ? d : d - half, c, s);
            r.c[i] = c[0], r.s[i] = d < half ? -s[0] : s[0];
        }
    }
}

// A row on its way: this lane's channels and their partners.
template <int TYPE> struct Raw {
    Elem8<TYPE> x, z;
};

template <int TYPE>
__device__ __forceinline__ void fetch(const PgWriteArgs &a, const Turn &T, Raw<TYPE> &r, const void *p, int64_t at, int d0)
{
    r.x = load8<TYPE>(p, at + d0, a.vec);
    if (T.on == 0 || !a.rot.halves) return;
    if ((a.rot.half & 7) == 0) {
        r.z = load8<TYPE>(p, at + T.e0, a.vec);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int d = min(d0 + i, 2 * a.rot.half - 1);
            r.z[i] = ((const typename Elem<TYPE>::type *)p)[at + (d < a.rot.half ? d + a.rot.half : d - a.rot.half)];
        }
    }
}

// The row normed and turned.  gamma: the norm's weights in LDS, head_dim of them and more.
template <int TYPE>
__device__ __forceinline__ void finish(const PgWriteArgs &a, const Turn &T, const float *gamma, const Raw<TYPE> &r, bool norm, int d0, float (&y)[8])
{
    float f = 1.0f;
    if (norm) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) sq = __builtin_fmaf((float)r.x[i], (float)r.x[i], sq);
        sq = row_sum(sq, a.group_shift);
        f = 1.0f / sqrtf(sq / (float)a.hd + a.eps);
    }
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = norm ? (float)r.x[i] * f * gamma[d0 + i] : (float)r.x[i];
    if (a.rot.halves && norm && (a.rot.half & 7) == 0) {
        const int e0 = T.on ? T.e0 : 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float w = (float)r.z[i] * f * gamma[e0 + i];
            y[i] = i < T.on ? x[i] * T.c[i] + w * T.s[i] : x[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) {
        float w = x[i ^ 1];
        if (a.rot.halves) {
            const int d = min(d0 + i, 2 * a.rot.half - 1);
            w = norm ? (float)r.z[i] * f * gamma[d < a.rot.half ? d + a.rot.half : d - a.rot.half] : (float)r.z[i];
        }
        y[i] = i < T.on ? x[i] * T.c[i] + w * T.s[i] : x[i];
    }
}

// A wave takes rows `part`, `part + splits` .. (64 >> group_shift at a time) of one token: the query heads, then the KV heads.
template <int TYPE>
__global__ __launch_bounds__(256) void k_paged_write(const PgWriteArgs a)
{
    __shared__ __align__(16) float gamma[2][kPgMaxHead];
    if ((int)threadIdx.x < a.hd) {
        gamma[0][threadIdx.x] = a.q_gamma ? a.q_gamma[threadIdx.x] : 1.0f;
        gamma[1][threadIdx.x] = a.k_gamma ? a.k_gamma[threadIdx.x] : 1.0f;
    }
    __syncthreads();
    const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int t = wave / a.splits, part = wave - t * a.splits;
    if (t >= a.n_tok) return;
    const int rows = 64 >> a.group_shift, lane = threadIdx.x & ((1 << a.group_shift) - 1), sub = (threadIdx.x & 63) >> a.group_shift;
    const int d0 = lane * 8, nq = a.q ? a.n_head : 0, items = nq + (a.k ? a.n_kv : 0);
    const bool on = d0 < a.hd;
    const int place = a.c.base ? a.places[t] : 0;
    const bool there = !a.c.base || (place >= 0 && place < a.c.n_pages * a.c.page);
    Turn T = turn_of(a, on ? d0 : a.hd);

    // two turns ahead
    struct Row {
        Raw<TYPE> r;
        Elem8<TYPE> v;
    } ahead[2] = {};
    const auto load = [&](Row &w, int g) {
        if (!on || g >= items) return;
        if (g < nq) {
            fetch<TYPE>(a, T, w.r, a.q, t * a.q_stride + (int64_t)g * a.hd, d0);
        } else {
            const int64_t h = (int64_t)(g - nq) * a.hd;
            fetch<TYPE>(a, T, w.r, a.k, t * a.k_stride + h, d0);
            if (a.c.base) w.v = load8<TYPE>(a.v, t * a.v_stride + h + d0, a.vec);
        }
    };
    const int step = a.splits * rows, g0 = part * rows + sub;
    load(ahead[0], g0);
    load(ahead[1], g0 + step);
    angles_of(a, T, t, d0);
    for (int g = g0; g < items; g += step) {
        const Raw<TYPE> cur = ahead[0].r;
        const Elem8<TYPE> cv = ahead[0].v;
        ahead[0] = ahead[1];
        load(ahead[1], g + 2 * step);
        float y[8];
        if (g < nq) {
            finish<TYPE>(a, T, gamma[0], cur, a.q_gamma, d0, y);
            if (on) store8(a.out_type, a.q_out, ((int64_t)t * a.n_head + g) * a.hd + d0, y, a.vec);
            continue;
        }
        const int head = g - nq;
        finish<TYPE>(a, T, gamma[1], cur, a.k_gamma, d0, y);
        if (!a.c.base) {
            if (on) store8(a.out_type, a.k_out, ((int64_t)t * a.n_kv + head) * a.hd + d0, y, a.vec);
            continue;
        }
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = (float)cv[i];
        Unit ku = rounded(a.c.bf16, y), vu = rounded(a.c.bf16, w);
        const uint64_t bad = __ballot(on && (ku.bad || vu.bad)) >> (sub << a.group_shift);   // this row's lanes lowest
        if (!on || !there) continue;
        if (bad & ((UINT64_C(1) << (1 << a.group_shift)) - 1)) {
            ku.u = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
            vu.u = make_uint4(0, 0, 0, 0);
        }
        const int p = place & (a.c.page - 1);
        uint8_t *row = a.c.k_row(place / a.c.page, head, p) + 16 * pg_unit(a.c.w, lane, p);
        *(uint4 *)row = ku.u;
        *(uint4 *)(row + a.c.v_off()) = vu.u;
    }
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
    // a token's rows over several waves where tokens are fewer than what keeps the chip busy (16 waves a compute unit)
    const int items = (a.q ? a.n_head : 0) + (a.k ? a.n_kv : 0), rows = 64 >> a.group_shift, turns = (items + rows - 1) / rows;
    a.splits = std::max(1, std::min(turns, 4096 / a.n_tok));
    const unsigned blocks = (unsigned)(((int64_t)a.n_tok * a.splits + 3) / 4);
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
