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
//
// What bounds it.  Memory (16383 tokens, 32 + 8 + 8 heads of 128, bf16: 95 to 100 us for 403 MB, 4.0 to 4.2 TB/s, where a large
// copy reaches 4.9; reading back 134 MB 21.7 us; queries and keys without a cache 86 us for 336 MB).  Few tokens: the chain from position to angle to row (16 tokens, 32 + 4 + 4
// heads of 64: 5.6 us).  bf16 rows leave registers for four waves on a SIMD; with three the first takes 13 us more.
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
    uint32_t w[4], over = 0;
    const uint32_t top = bf16 ? 0x7F807F80u : 0x7C007C00u, least = bf16 ? 0x00800080u : 0x04000400u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        typedef _Float16 half2v __attribute__((ext_vector_type(2)));
        w[i] = bf16 ? bf16_pair(x[2 * i], x[2 * i + 1]) : __builtin_bit_cast(uint32_t, half2v{(_Float16)x[2 * i], (_Float16)x[2 * i + 1]});
        over |= (w[i] & top) + least;   // an exponent of all ones carries into the sign's place
    }
    return Unit{make_uint4(w[0], w[1], w[2], w[3]), (over & 0x80008000u) != 0};
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

// What the lanes of a wave share about its token.
struct Token {
    Turn turn;
    int t, d0, first, step;   // this lane's channels; its first row, and how far to the next one
    bool on;                  // the lane has channels
};

// One kind of rows of a token: queries, or keys with their values (KV).  put(row, y, v): the row normed and turned, its V row.
// x f A + z f B with A = gamma c and B = gamma' s: the norm's factor f first, since x gamma may leave fp32 where x f gamma does not.
template <int TYPE, bool VEC, bool KV, typename Put>
__device__ __forceinline__ void each_row(const PgWriteArgs &a, const Token &k, const void *src, const void *vsrc, int rows, const float *gamma,
                                         bool norm, Put put)
{
    typedef typename Elem<TYPE>::type E;
    const Turn &T = k.turn;
    const int half = a.rot.half, d0 = k.d0;
    const bool halves = a.rot.halves, apart = halves && (half & 7) != 0, partial = 2 * half < a.hd;
    float A[8], B[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int d = min(d0 + i, max(2 * half - 1, 0)), e = halves ? (d < half ? d + half : d - half) : d ^ 1;
        A[i] = (norm ? gamma[d0 + i] : 1.0f) * (i < T.on ? T.c[i] : 1.0f);
        B[i] = i < T.on ? (norm ? gamma[e] : 1.0f) * T.s[i] : 0.0f;
    }
    struct Raw {
        Elem8<TYPE> x, z, v;
    };
    const E *x = (const E *)src + (int64_t)k.first * a.hd;
    const int64_t to_v = KV ? (const uint8_t *)vsrc - (const uint8_t *)src : 0;
    const int64_t stride = (int64_t)k.step * a.hd;
    const auto load = [&](Raw &r, int g) {
        if (k.on && g < rows) {
            r.x = load8<TYPE>(x, d0, VEC);
            if (apart) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int d = min(d0 + i, 2 * half - 1);
                    r.z[i] = x[d < half ? d + half : d - half];
                }
            } else if (halves && T.on) {
                r.z = load8<TYPE>(x, T.e0, VEC);
            }
            if (KV) r.v = load8<TYPE>((const uint8_t *)x + to_v, d0, VEC);
        }
        x += stride;
    };
    Raw ahead[2] = {};   // two turns ahead
    load(ahead[0], k.first);
    load(ahead[1], k.first + k.step);
    for (int g = k.first; g < rows; g += k.step) {
        const Raw r = ahead[0];
        ahead[0] = ahead[1];
        load(ahead[1], g + 2 * k.step);
        float y[8], xs[8], zs[8];
#pragma unroll
        for (int i = 0; i < 8; i++) xs[i] = (float)r.x[i], zs[i] = halves ? (float)r.z[i] : 0.0f;
        if (norm) {
            float sq = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) sq = __builtin_fmaf(xs[i], xs[i], sq);
            const float m = row_sum(sq, a.group_shift) * a.inv_hd + a.eps;
            float f = __builtin_amdgcn_rsqf(m);
            // squares that leave fp32 (fp16's do not, but the least eps beside zeros does): again, with a power of two
            const bool far = !(m >= 1.17549435e-38f && m < __builtin_huge_valf());
            if (__any(far)) {
                const float by = m < 1.0f ? 0x1p96f : 0x1p-72f;
                // (from memory, one by one: few registers for what hardly ever happens)
                const E *p = x - 3 * stride + d0;
                sq = 0.0f;
#pragma unroll 1
                for (int i = 0; k.on && i < 8; i++) {
                    const float w = (float)p[i] * by;
                    sq = __builtin_fmaf(w, w, sq);
                }
                const float root = 1.0f / sqrtf(row_sum(sq, a.group_shift) * a.inv_hd + a.eps * by * by);
                // x by root, in the order that leaves no product outside: small rows times `by` first, large ones last
                const float last = !far ? 1.0f : m < 1.0f ? root : by;
                if (far) f = m < 1.0f ? by : root;
#pragma unroll
                for (int i = 0; i < 8; i++) xs[i] *= f, zs[i] *= f;
                f = last;
            }
#pragma unroll
            for (int i = 0; i < 8; i++) xs[i] *= f, zs[i] *= f;
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            float z = halves ? zs[i] : xs[i ^ 1];
            if (partial) z = i < T.on ? z : 0.0f;
            y[i] = __builtin_fmaf(z, B[i], xs[i] * A[i]);
        }
        put(g, y, r.v);
    }
}

// A wave takes rows `part`, `part + splits` .. (64 >> group_shift at a time) of one token, queries, then keys and values; with
// q_parts > 0 only queries, or (from part q_parts on) only keys and values.
template <int TYPE, bool VEC>
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
    Token k;
    k.t = t, k.d0 = lane * 8, k.on = k.d0 < a.hd;
    const bool only_q = part < a.q_parts, only_kv = a.q_parts > 0 && !only_q;
    const int own = only_kv ? part - a.q_parts : part, of = only_q ? a.q_parts : a.splits - a.q_parts;
    k.first = own * rows + sub, k.step = of * rows;
    k.turn = turn_of(a, k.on ? k.d0 : a.hd);
    angles_of(a, k.turn, t, k.d0);
    if (!k.on) k.d0 = 0;   // (never more than is there)
    typedef typename Elem<TYPE>::type E;
    if (a.q && !only_kv)
        each_row<TYPE, VEC, false>(a, k, (const E *)a.q + t * a.q_stride, nullptr, a.n_head, gamma[0], a.q_gamma, [&](int g, const float (&y)[8], auto) {
            if (k.on) store8(a.out_type, a.q_out, ((int64_t)t * a.n_head + g) * a.hd + k.d0, y, VEC);
        });
    if (!a.k || only_q) return;
    const E *src = (const E *)a.k + t * a.k_stride;
    if (!a.c.base) {
        each_row<TYPE, VEC, false>(a, k, src, nullptr, a.n_kv, gamma[1], a.k_gamma, [&](int g, const float (&y)[8], auto) {
            if (k.on) store8(a.out_type, a.k_out, ((int64_t)t * a.n_kv + g) * a.hd + k.d0, y, VEC);
        });
        return;
    }
    const int place = a.places[t];
    if (place < 0 || place >= a.c.n_pages * a.c.page) return;
    const int p = place & (a.c.page - 1);
    uint8_t *to = a.c.k_row(place / a.c.page, 0, p) + 16 * pg_unit(a.c.w, lane, p);
    each_row<TYPE, VEC, true>(a, k, src, (const E *)a.v + t * a.v_stride, a.n_kv, gamma[1], a.k_gamma, [&](int g, const float (&y)[8], Elem8<TYPE> v) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; i++) w[i] = (float)v[i];
        Unit ku = rounded(a.c.bf16, y), vu = rounded(a.c.bf16, w);
        const uint64_t bad = __ballot(k.on && (ku.bad || vu.bad)) >> (sub << a.group_shift);   // this row's lanes lowest
        if (!k.on) return;
        if (bad & ((UINT64_C(1) << (1 << a.group_shift)) - 1)) {
            ku.u = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
            vu.u = make_uint4(0, 0, 0, 0);
        }
        uint8_t *row = to + g * a.c.head_bytes();
        *(uint4 *)row = ku.u;
        *(uint4 *)(row + a.c.v_off()) = vu.u;
    });
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
    // and each kind of them over waves of its own where that still leaves every row its turn at once (16 tokens of 32 + 4 heads of
    // 64: 5.4 us for 7.3)
    const int rows = 64 >> a.group_shift, tq = ((a.q ? a.n_head : 0) + rows - 1) / rows, tk = ((a.k ? a.n_kv : 0) + rows - 1) / rows;
    const bool apart = tq > 0 && tk > 0 && (int64_t)a.n_tok * (tq + tk) <= 4096;
    a.q_parts = apart ? tq : 0;
    a.splits = apart ? tq + tk : std::max(1, std::min(std::max(tq, tk), 4096 / a.n_tok));
    const unsigned blocks = (unsigned)(((int64_t)a.n_tok * a.splits + 3) / 4);
    a.inv_hd = 1.0f / (float)a.hd;
    if (in_type == PG_F32 && a.vec) k_paged_write<PG_F32, true><<<blocks, 256, 0, s>>>(a);
    else if (in_type == PG_F32) k_paged_write<PG_F32, false><<<blocks, 256, 0, s>>>(a);
    else if (in_type == PG_F16 && a.vec) k_paged_write<PG_F16, true><<<blocks, 256, 0, s>>>(a);
    else if (in_type == PG_F16) k_paged_write<PG_F16, false><<<blocks, 256, 0, s>>>(a);
    else if (a.vec) k_paged_write<PG_BF16, true><<<blocks, 256, 0, s>>>(a);
    else k_paged_write<PG_BF16, false><<<blocks, 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_paged_read(const PgView &c, const int32_t *places, int n_tok, void *k, void *v, hipStream_t s)
{
    const int64_t n = (int64_t)n_tok * c.n_kv * (c.hd / 8);
    k_paged_read<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(c, places, n_tok, (uint16_t *)k, (uint16_t *)v);
    return hipGetLastError();
}

}  // namespace smx
