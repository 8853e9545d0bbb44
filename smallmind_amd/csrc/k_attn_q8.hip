// k_attn_q8.hip -- attention of a batch of sequences over the 8-bit KV cache (smx_kvcache.h): n_q new
// tokens of every sequence against the positions of its own slot, and, with a prefix, against a slot
// that the whole batch shares.
//
// Mathematics.  A row is one query head of one token, its KV head's cache holds codes k, v in
// [-127, 127] with scales a_p, b_p per position p.  With x_p = a_p (q . k_p), c = log2(e) / sqrt(hd) and
// the running maximum m of x,
//     out = sum_p 2^(c (x_p - m)) b_p v_p / sum_p 2^(c (x_p - m)),
// one pass over the positions, in tiles of 64.  The scales stay out of the products, so these take the
// codes themselves, which fp16 holds exactly.  The other operands, q and w_p = 2^(c (x_p - m)) b_p, go
// in as two fp16 values each, high part and remainder, both rounded to nearest, after a power of two has
// brought the largest of the row (of q) or of the scales (b) below 2^15: 22 bits of every value down to
// 2^-28 of the largest, 2^-39 of it in absolute terms, against the 24 bits of fp32; sums are fp32.
// (One fp16 part would leave 11 bits: errors of 1e-4 where the fp32 outputs should have 1e-6.  bf16 parts
// need three, and half as much again of the matrix instructions.)
//
// Layout.  A wave computes S^T = K q^T on 16x16x32 matrix instructions: lane 16 g + c gets
// row c's x at positions 16 t + 4 g + i, which is how the second product out^T = V^T w^T wants them, so the
// weights go from one product to the next without moving between lanes, and a row's maximum and sum
// need two lane exchanges.  The contraction order of q K^T is whatever 16-byte loads give.
//
// Two ways through the positions, cut into chunks of one workgroup each; k_attn_q8_join adds up what the
// chunks found.
//   stream: few rows per KV head (a sequence's own positions, where reading them is what takes time).  All
//           four waves hold the same 16 rows and take tiles in turn, each from memory to registers;
//           they join their sums through LDS at the end.  K of the next tile is requested as soon as
//           this tile's products have used it, V likewise.
//   rows:   many rows per KV head (a prefix that many sequences share, where the arithmetic is what
//           takes time).  Every wave holds 16 or 32 rows of its own, and all walk the same tiles, which the
//           workgroup turns into fp16 once and keeps in LDS in the order of the matrix instructions' lanes.
#include <type_traits>

#include "smx_attn_q8.h"
#include "smx_device.h"
#include "smx_internal.h"

#ifndef SMX_ATTN_W
#error "SMX_ATTN_W: the cache's row width"
#endif

namespace smx {

namespace {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

constexpr int W = SMX_ATTN_W;
constexpr int NC = W / 64;               // 64-wide pieces of a K row: 16 bytes per lane
constexpr bool TAIL = W % 64 != 0;       // and a 32-wide one: 8 bytes per lane
constexpr int NK = W / 32;               // matrix instructions along a K row
constexpr int ND = W / 16;               // 16-dim groups of the output
constexpr int NW = 4;                    // waves of a workgroup
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLeast = 7.8886090522101181e-31f;   // 2^-100: no power of two below it is used as a scale

__device__ __forceinline__ half8 halves(uint32_t lo, uint32_t hi)
{
    // byte b under the high byte 0x64 is the fp16 1024 + b; 1024 + 128 less is the code
    union { uint32_t u[4]; half2v h[4]; half8 v; } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
    const half2v z = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int i = 0; i < 4; i++) r.h[i] = r.h[i] - z;
    return r.v;
}

// The power of two 2^e with 2^(e-1) < f <= 2^e (f finite and positive).
__device__ __forceinline__ float pow2_above(float f)
{
    return __uint_as_float((__float_as_uint(f) + 0x7FFFFFu) & 0x7F800000u);
}

// Two values as fp16 parts: h the nearest, l what is left.
__device__ __forceinline__ void split(float a, float b, half2v &h, half2v &l)
{
    h = half2v{(_Float16)a, (_Float16)b};
    l = half2v{(_Float16)__builtin_fmaf((float)h[0], -1.0f, a), (_Float16)__builtin_fmaf((float)h[1], -1.0f, b)};
}

__device__ __forceinline__ void put(half8 &v, int at, half2v h) { v[at] = h[0], v[at + 1] = h[1]; }

__device__ __forceinline__ float max_groups(float v)   // over the four lanes of a column
{
    float2 p = swap32(v, v);
    v = fmaxf(p.x, p.y);
    p = swap16(v, v);
    return fmaxf(p.x, p.y);
}

__device__ __forceinline__ float max_lanes(float v)   // over the wave
{
    v = fmaxf(v, dpp_mov<0xB1>(v));
    v = fmaxf(v, dpp_mov<0x4E>(v));
    v = fmaxf(v, dpp_mov<0x141>(v));
    v = fmaxf(v, dpp_mov<0x140>(v));
    return max_groups(v);
}

__device__ __forceinline__ float sum_groups(float v)
{
    float2 p = swap32(v, v);
    v = p.x + p.y;
    p = swap16(v, v);
    return p.x + p.y;
}

// Keeps the compiler from moving instructions across: without it, it fetches all operands of a tile before
// the first product and runs out of registers.
__device__ __forceinline__ void here() { __builtin_amdgcn_sched_barrier(0); }

struct KTile {
    uint4v a[4][NC > 0 ? NC : 1];
    uint2v b[4];
};
struct VTile {
    uint4v a[ND];
};

__device__ __forceinline__ void load_k(KTile &k, const uint8_t *rec, int g, int col)
{
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint8_t *p = rec + (16 * t + col) * W;
#pragma unroll
        for (int n = 0; n < NC; n++) k.a[t][n] = *(const uint4v *)(p + 64 * n + 16 * g);
        if constexpr (TAIL) k.b[t] = *(const uint2v *)(p + 64 * NC + 8 * g);
    }
}

__device__ __forceinline__ void load_v(VTile &v, const uint8_t *rec, int g, int col)
{
    const uint8_t *p = rec + kKvTile * W + col * kKvTile + 16 * g;
#pragma unroll
    for (int n = 0; n < ND; n++) v.a[n] = *(const uint4v *)(p + 16 * kKvTile * n);
}

struct RowRef {          // a row of the batch
    bool valid;
    int token, head;     // token: sequence * n_q + i
};

// Joining of a workgroup's NW waves' sums.
struct Shared {
    float m[NW][16], l[NW][16];
    float acc[NW][16][W + 4];
};

// The rows' queries as the second operands of K q^T, and c in the units of their products.
template <int MT, typename RowOf>
__device__ __forceinline__ void load_q(const AttnQ8Args &a, half8 (&qh)[MT][NK], half8 (&ql)[MT][NK], float (&c)[MT], int g,
                                       int col, RowOf row_of)
{
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const RowRef r = row_of(16 * mt + col);
        const float *q = a.q + (int64_t)r.token * a.q_stride + (int64_t)r.head * a.hd;
        float f[NK][8];
        uint32_t top = 0;
#pragma unroll
        for (int n = 0; n < NK; n++) {
            // the dims of this lane's bytes: 16 g + 8 (n % 2) of piece n / 2, 8 g of the 32-wide one
            const int d = TAIL && n == NK - 1 ? 64 * NC + 8 * g : 64 * (n >> 1) + 16 * g + 8 * (n & 1);
            const bool in = r.valid && d < a.hd;   // head_dim is a multiple of 8
            if (a.q_vec) {
                float4v u = {0, 0, 0, 0}, v = {0, 0, 0, 0};
                if (in) u = *(const float4v *)(q + d), v = *(const float4v *)(q + d + 4);
#pragma unroll
                for (int e = 0; e < 4; e++) f[n][e] = u[e], f[n][4 + e] = v[e];
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) f[n][e] = in ? q[d + e] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(f[n][e]) & 0x7FFFFFFFu);
        }
        const float amax = max_groups(__uint_as_float(min(top, 0x7F7FFFFFu)));
        const bool bad = max_groups(top > 0x7F7FFFFFu ? 1.0f : 0.0f) > 0.0f;   // a NaN or infinity: the row is NaN
        const float unit = amax > kLeast ? __uint_as_float(__float_as_uint(amax) & 0x7F800000u) : kLeast;   // 2^e
        const float mul = bad ? __uint_as_float(0x7FC00000u) : __uint_as_float((268u << 23) - __float_as_uint(unit));   // 2^14 / unit
        c[mt] = a.scale_log2e * (unit * (1.0f / 16384.0f));
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                half2v h, l;
                split(f[n][e] * mul, f[n][e + 1] * mul, h, l);
                put(qh[mt][n], e, h);
                put(ql[mt][n], e, l);
            }
    }
}

// x = K q^T of a tile; k_of(t, n): the codes of positions 16 t .. as operand n along the row.  The operands of
// the next n are made ready beside the products of this one; the products of four position groups lie
// between two that add to the same sum.
template <int MT, typename KOf>
__device__ __forceinline__ void scores(float4v (&x)[MT][4], const half8 (&qh)[MT][NK], const half8 (&ql)[MT][NK], KOf k_of)
{
    half8 k[2][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        k[0][t] = k_of(t, 0);
#pragma unroll
        for (int mt = 0; mt < MT; mt++) x[mt][t] = float4v{0, 0, 0, 0};
    }
#pragma unroll
    for (int n = 0; n < NK; n++) {
        if (n + 1 < NK) {
#pragma unroll
            for (int t = 0; t < 4; t++) k[(n + 1) & 1][t] = k_of(t, n + 1);
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                x[mt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[n & 1][t], qh[mt][n], x[mt][t], 0, 0, 0);
#pragma unroll
        for (int mt = 0; mt < MT; mt++)
#pragma unroll
            for (int t = 0; t < 4; t++)
                x[mt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[n & 1][t], ql[mt][n], x[mt][t], 0, 0, 0);
        here();
    }
}

// acc += V^T w^T of a tile; v_of(n, kb): the codes of dims 16 n .. at the positions of half kb.  Two groups
// of dims at a time, the next two made ready beside their products.
template <int MT, typename VOf>
__device__ __forceinline__ void weigh(float4v (&acc)[MT][ND], const half8 (&ph)[MT][2], const half8 (&pl)[MT][2], VOf v_of)
{
    half8 v[2][2][2];
#pragma unroll
    for (int j = 0; j < 4; j++) v[0][j >> 1][j & 1] = v_of(j >> 1, j & 1);
#pragma unroll
    for (int n0 = 0; n0 < ND; n0 += 2) {   // (ND is even)
        const int b = (n0 >> 1) & 1;
        if (n0 + 2 < ND) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[b ^ 1][j >> 1][j & 1] = v_of(n0 + 2 + (j >> 1), j & 1);
        }
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++)
                    acc[mt][n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b][n][kb], ph[mt][kb], acc[mt][n0 + n], 0, 0, 0);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int n = 0; n < 2; n++)
                    acc[mt][n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b][n][kb], pl[mt][kb], acc[mt][n0 + n], 0, 0, 0);
        }
        here();
    }
}

// The running softmax of MT blocks of rows.
template <int MT>
struct Running {
    // m: the largest x so far; mc: c m as rounded, the exponent that acc and l are relative to
    float m[MT], mc[MT], l[MT], c[MT];
    float vref;   // power of two, at least every V scale so far: acc is relative to 2^-14 of it
    float4v acc[MT][ND];

    __device__ __forceinline__ void clear()
    {
        vref = kLeast;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            m[mt] = mc[mt] = kNegInf;
            l[mt] = 0.0f;
#pragma unroll
            for (int n = 0; n < ND; n++) acc[mt][n] = float4v{0, 0, 0, 0};
        }
    }

    // One tile: x (K q^T) becomes the weights' parts, acc and l move to the new maximum.  ks(t), vs(t): the
    // scales of this lane's positions, vone: the V scale of position `lane`.  With WHOLE every position counts
    // for every row; otherwise the tile's first `left` exist and row block mt sees its first vis[mt]; what is
    // not seen weighs nothing whatever its scales hold.
    template <bool WHOLE, typename KsOf, typename VsOf>
    __device__ __forceinline__ void step(float4v (&x)[MT][4], KsOf ks, VsOf vs, float vone, half8 (&ph)[MT][2],
                                         half8 (&pl)[MT][2], int left, const int (&vis)[MT], int lane)
    {
        const int g = lane >> 4;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float4v k = ks(t);
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                x[mt][t] *= k;
                if constexpr (!WHOLE) {
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (16 * t + 4 * g + i >= vis[mt]) x[mt][t][i] = kNegInf;
                }
            }
        }
        if (!WHOLE && lane >= left) vone = 0.0f;
        const float vnew = fmaxf(vref, pow2_above(max_lanes(fmaxf(vone, kLeast))));
        const float vmul = __uint_as_float((268u << 23) - __float_as_uint(vnew));   // 2^14 / vnew
        const float vdown = vref * (vmul * (1.0f / 16384.0f));
        vref = vnew;
        float now[MT], sum[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float top = m[mt];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, x[mt][t][i]);
            top = max_groups(top);
            // (a row that has seen nothing yet: x = -inf against 0)
            now[mt] = top == kNegInf ? 0.0f : top * c[mt];
            const float alpha = __builtin_amdgcn_exp2f(mc[mt] - now[mt]);
            if (top != kNegInf) m[mt] = top, mc[mt] = now[mt];
            l[mt] *= alpha;
            sum[mt] = 0.0f;
            const float down = alpha * vdown;
            if (__any(down != 1.0f)) {
#pragma unroll
                for (int n = 0; n < ND; n++) acc[mt][n] *= down;
            }
        }
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float4v v = vs(t) * vmul;
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[mt][t][i], c[mt], -now[mt]));
                    sum[mt] += p;
                    w[i] = p * v[i];
                    if (!WHOLE && 16 * t + 4 * g + i >= vis[mt]) w[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    half2v h, r;
                    split(w[i], w[i + 1], h, r);
                    put(ph[mt][t >> 1], 4 * (t & 1) + i, h);
                    put(pl[mt][t >> 1], 4 * (t & 1) + i, r);
                }
            }
            here();
        }
#pragma unroll
        for (int mt = 0; mt < MT; mt++) l[mt] += sum[mt];
    }
};

// stream: the NW waves take the tiles of positions [p0, p1) in turn; vis_of(row): positions that the row
// sees, counted from the slot's first, min_vis at least.
template <typename RowOf, typename VisOf>
__device__ __forceinline__ void stream(const AttnQ8Args &a, Shared &S, const uint8_t *cache, int p0, int p1, int min_vis,
                                       RowOf row_of, VisOf vis_of)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, wave = wave_id();
    const int n_tiles = (p1 - p0 + kKvTile - 1) / kKvTile;
    constexpr size_t REC = kv_tile_bytes(W);

    const uint8_t *rec = cache + (size_t)(p0 / kKvTile + wave) * REC;
    KTile kt;
    VTile vt;
    if (wave < n_tiles) {
        load_k(kt, rec, g, col);
        load_v(vt, rec, g, col);
    }
    half8 qh[1][NK], ql[1][NK];
    Running<1> R;
    R.clear();
    load_q<1>(a, qh, ql, R.c, g, col, row_of);
    const int vis = row_of(col).valid ? vis_of(col) : 0;

    // tiles that every row sees all of, then the rest: the same code with and without the bounds
    const auto go = [&](int &tile, int end, auto whole) {
        for (; tile < end; tile += NW) {
            const float *scales = (const float *)(rec + 2 * kKvTile * W);
            float4v ks[4], vs[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                ks[t] = *(const float4v *)(scales + 16 * t + 4 * g);
                vs[t] = *(const float4v *)(scales + kKvTile + 16 * t + 4 * g);
            }
            const float vone = scales[kKvTile + lane];
            rec += NW * REC;
            const bool more = tile + NW < n_tiles;
            float4v x[1][4];
            scores<1>(x, qh, ql, [&](int t, int n) {
                if (TAIL && n == NK - 1) return halves(kt.b[t][0], kt.b[t][1]);
                return halves(kt.a[t][n >> 1][2 * (n & 1)], kt.a[t][n >> 1][2 * (n & 1) + 1]);
            });
            if (more) load_k(kt, rec, g, col);
            const int at = p0 + tile * kKvTile;
            const int seen[1] = {vis - at};
            half8 ph[1][2], pl[1][2];
            R.template step<decltype(whole)::value>(
                x, [&](int t) { return ks[t]; }, [&](int t) { return vs[t]; }, vone, ph, pl, p1 - at, seen, lane);
            weigh<1>(R.acc, ph, pl, [&](int n, int kb) { return halves(vt.a[n][2 * kb], vt.a[n][2 * kb + 1]); });
            if (more) load_v(vt, rec, g, col);
        }
    };
    int tile = wave;
    go(tile, min(n_tiles, (min_vis - p0) / kKvTile), std::true_type{});
    go(tile, n_tiles, std::false_type{});

    const float sum = sum_groups(R.l[0]), up = R.vref * (1.0f / 16384.0f);
    if (g == 0) {
        S.m[wave][col] = R.mc[0];
        S.l[wave][col] = sum;
    }
#pragma unroll
    for (int n = 0; n < ND; n++) *(float4v *)&S.acc[wave][col][16 * n + 4 * g] = R.acc[0][n] * up;
    __syncthreads();
}

// Joins the waves' sums and writes the rows: the outputs, or with more parts to come the part's
// maximum (in powers of two), sum and weighted sums.
template <typename RowOf>
__device__ __forceinline__ void finish(const AttnQ8Args &a, Shared &S, int part, RowOf row_of)
{
    for (int i = threadIdx.x; i < 16 * (W / 4); i += 64 * NW) {
        const int row = i / (W / 4), d = 4 * (i % (W / 4));
        const RowRef r = row_of(row);
        if (!r.valid || d >= a.hd) continue;
        float top = kNegInf, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) top = fmaxf(top, S.m[w][row]);
        float4v o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            // a wave without a visible position has the sum 0 (and one that saw NaN a NaN)
            const float f = S.m[w][row] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(S.m[w][row] - top);
            if (S.l[w][row] == 0.0f) continue;
            sum += S.l[w][row] * f;
            o += *(const float4v *)&S.acc[w][row][d] * f;
        }
        const int64_t id = (int64_t)r.token * a.n_head + r.head;
        if (a.direct) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            float *dst = a.out + id * a.hd + d;
            if (a.out_vec) {
                *(float4v *)dst = o * inv;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) dst[e] = o[e] * inv;
            }
        } else {
            float *ml = a.part_ml + (part * a.n_rows + id) * 2;
            if (d == 0) ml[0] = top, ml[1] = sum;
            *(float4v *)(a.part_acc + (part * a.n_rows + id) * a.hd + d) = o;
        }
    }
}

// rows: the tiles as fp16 operands in LDS, in fragments of 1 KB, a lane's 16 bytes after another's: K by (t, n),
// V by (n, kb).  A second buffer takes the next tile while this one is read, where there is room.
constexpr int NB = W <= 128 ? 2 : 1;
struct Tiles {
    half8 k[NB][4][NK][64], v[NB][ND][2][64];
    float scale[NB][2][kKvTile];
};

// Positions [p0, p1), all seen by every row; the workgroup's wave w has the rows row_of(0 .. 16 MT - 1).
// Writes the rows' part.
template <int MT, typename RowOf>
__device__ __forceinline__ void rows(const AttnQ8Args &a, Tiles &S, const uint8_t *cache, int p0, int p1, int part, RowOf row_of)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, wave = wave_id();
    const int n_tiles = (p1 - p0 + kKvTile - 1) / kKvTile;
    constexpr size_t REC = kv_tile_bytes(W);
    constexpr int NV = (ND + 3) / 4;   // V groups that a wave brings in

    half8 qh[MT][NK], ql[MT][NK];
    Running<MT> R;
    R.clear();
    load_q<MT>(a, qh, ql, R.c, g, col, row_of);
    const bool busy = __any(row_of(0).valid);

    // this wave's share of a tile: K of positions 16 wave .., V of dims 16 (wave + 4 j) ..
    uint4v ka[NC > 0 ? NC : 1], va[NV];
    uint2v kb2;
    float sc = 0.0f;
    const auto load = [&](const uint8_t *rec) {
        const uint8_t *k = rec + (16 * wave + col) * W, *v = rec + kKvTile * W + col * kKvTile + 16 * g;
#pragma unroll
        for (int n = 0; n < NC; n++) ka[n] = *(const uint4v *)(k + 64 * n + 16 * g);
        if constexpr (TAIL) kb2 = *(const uint2v *)(k + 64 * NC + 8 * g);
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (wave + 4 * j < ND) va[j] = *(const uint4v *)(v + 16 * kKvTile * (wave + 4 * j));
        if (threadIdx.x < 2 * kKvTile) sc = ((const float *)(rec + 2 * kKvTile * W))[threadIdx.x];
    };
    const uint8_t *rec = cache + (size_t)(p0 / kKvTile) * REC;
    load(rec);
    const auto go = [&](int &tile, int end, auto whole) {
        for (; tile < end; tile++) {
            const int b = NB == 2 ? tile & 1 : 0;
            if (NB == 1 && tile > 0) __syncthreads();   // the tile before has been read
#pragma unroll
            for (int n = 0; n < NC; n++) {
                S.k[b][wave][2 * n][lane] = halves(ka[n][0], ka[n][1]);
                S.k[b][wave][2 * n + 1][lane] = halves(ka[n][2], ka[n][3]);
            }
            if constexpr (TAIL) S.k[b][wave][NK - 1][lane] = halves(kb2[0], kb2[1]);
#pragma unroll
            for (int j = 0; j < NV; j++)
                if (wave + 4 * j < ND) {
                    S.v[b][wave + 4 * j][0][lane] = halves(va[j][0], va[j][1]);
                    S.v[b][wave + 4 * j][1][lane] = halves(va[j][2], va[j][3]);
                }
            if (threadIdx.x < 2 * kKvTile) S.scale[b][threadIdx.x >> 6][threadIdx.x & 63] = sc;
            rec += REC;
            if (tile + 1 < n_tiles) load(rec);
            __syncthreads();
            if (!busy) continue;
            float4v x[MT][4];
            scores<MT>(x, qh, ql, [&](int t, int n) { return S.k[b][t][n][lane]; });
            const int left = p1 - p0 - tile * kKvTile;
            int seen[MT];
#pragma unroll
            for (int mt = 0; mt < MT; mt++) seen[mt] = left;
            half8 ph[MT][2], pl[MT][2];
            R.template step<decltype(whole)::value>(
                x, [&](int t) { return *(const float4v *)&S.scale[b][0][16 * t + 4 * g]; },
                [&](int t) { return *(const float4v *)&S.scale[b][1][16 * t + 4 * g]; }, S.scale[b][1][lane], ph, pl, left, seen, lane);
            weigh<MT>(R.acc, ph, pl, [&](int n, int kb) { return S.v[b][n][kb][lane]; });
        }
    };
    int tile = 0;
    go(tile, (p1 - p0) / kKvTile, std::true_type{});
    go(tile, n_tiles, std::false_type{});
    if (!busy) return;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const RowRef r = row_of(16 * mt + col);
        const float sum = sum_groups(R.l[mt]), up = R.vref * (1.0f / 16384.0f);
        if (!r.valid) continue;
        const int64_t id = (int64_t)part * a.n_rows + (int64_t)r.token * a.n_head + r.head;
        if (g == 0) a.part_ml[id * 2] = R.mc[mt], a.part_ml[id * 2 + 1] = sum;
#pragma unroll
        for (int n = 0; n < ND; n++)
            if (16 * n + 4 * g < a.hd) *(float4v *)(a.part_acc + id * a.hd + 16 * n + 4 * g) = R.acc[mt][n] * up;
    }
}

// PRE, MTP: how the prefix is gone through, and 16-row blocks per wave there; the sequences' own positions:
// stream.
template <AttnQ8Pre PRE, int MTP>
__global__ __launch_bounds__(64 * NW, W <= 64 && MTP == 1 ? 3 : W <= 128 ? 2 : 1) void k_attn_q8(const AttnQ8Args a)
{
    union Mem {
        Shared own;
        std::conditional_t<PRE == PRE_ROWS, Tiles, int> tiles;
    };
    __shared__ __align__(16) char mem[sizeof(Mem)];
    Mem &S = *(Mem *)mem;
    const int group = a.n_head / a.n_kv;
    int b = blockIdx.x;
    if (PRE != PRE_NONE && b < a.pre_wgs) {
        // (chunk, KV head) fastest: workgroups that read the same positions are a multiple of 8 apart
        const int pairs = a.n_kv * a.pre_splits, pair = b % pairs, rb = b / pairs;
        const int head = pair % a.n_kv, split = pair / a.n_kv;
        const int p0 = split * a.pre_chunk, p1 = min(a.prefix_len, p0 + a.pre_chunk);
        const int row0 = PRE == PRE_ROWS ? (rb * 4 + wave_id()) * 16 * MTP : rb * 16, n_rows = a.n_seq * a.n_q * group;
        const auto row_of = [&](int r) {
            const int id = row0 + r;
            return RowRef{id < n_rows, id / group, head * group + id % group};
        };
        const uint8_t *cache = a.cache + (size_t)(a.prefix_slot * (int64_t)a.n_kv + head) * a.head_bytes;
        if constexpr (PRE == PRE_ROWS) {
            rows<MTP>(a, S.tiles, cache, p0, p1, split, row_of);
        } else {
            stream(a, S.own, cache, p0, p1, a.prefix_len, row_of, [&](int) { return a.prefix_len; });
            finish(a, S.own, split, row_of);
        }
        return;
    }
    b -= a.pre_wgs;
    const int pairs = a.n_seq * a.n_kv, pair = b % pairs;
    const int head = pair % a.n_kv, seq = pair / a.n_kv, rest = b / pairs;
    const int rb = rest % a.own_blocks, split = rest / a.own_blocks;
    const int slot = a.slots[seq];
    const bool active = (unsigned)slot < (unsigned)a.n_slots;
    const int len = active ? min(max(a.lens[seq], 0), a.max_len) : 0;
    const int p0 = split * a.own_chunk, p1 = min(len, p0 + a.own_chunk);
    const int row0 = rb * 16, n_rows = a.n_q * group;
    const auto row_of = [&](int r) {
        const int id = row0 + r;
        return RowRef{id < n_rows, seq * a.n_q + id / group, head * group + id % group};
    };
    const int part = a.pre_splits + split;
    if (p0 >= p1) {
        // nothing here: zeros, or a part without weight
        for (int i = threadIdx.x; i < 16 * W; i += 64 * NW) {
            const int row = i / W, d = i % W;
            const RowRef r = row_of(row);
            if (!r.valid || d >= a.hd) continue;
            const int64_t id = (int64_t)r.token * a.n_head + r.head;
            if (a.direct) {
                a.out[id * a.hd + d] = 0.0f;
            } else if (d == 0) {
                float *ml = a.part_ml + (part * a.n_rows + id) * 2;
                ml[0] = kNegInf, ml[1] = 0.0f;
            }
        }
        return;
    }
    // the first of the n_q tokens sees len - n_q + 1 positions, each further one sees one more
    stream(a, S.own, a.cache + (size_t)(slot * (int64_t)a.n_kv + head) * a.head_bytes, p0, p1, len - a.n_q + 1, row_of,
                [&](int r) { return len - a.n_q + 1 + (row0 + r) / group; });
    finish(a, S.own, part, row_of);
}

}  // namespace

#define SMX_LAUNCH_NAME_(w) launch_attn_q8_w##w
#define SMX_LAUNCH_NAME(w) SMX_LAUNCH_NAME_(w)
hipError_t SMX_LAUNCH_NAME(SMX_ATTN_W)(const AttnQ8Args &a, const AttnQ8Plan &p, hipStream_t s)
{
    const unsigned blocks = (unsigned)p.blocks;
    if (p.pre == PRE_NONE) k_attn_q8<PRE_NONE, 1><<<blocks, 64 * NW, 0, s>>>(a);
    else if (p.pre == PRE_STREAM) k_attn_q8<PRE_STREAM, 1><<<blocks, 64 * NW, 0, s>>>(a);
    else if (p.mt_pre == 1) k_attn_q8<PRE_ROWS, 1><<<blocks, 64 * NW, 0, s>>>(a);
    else if constexpr (kAttnQ8Narrow<SMX_ATTN_W>) k_attn_q8<PRE_ROWS, 2><<<blocks, 64 * NW, 0, s>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace smx
