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
// brought the row's largest below 2^15 (q) or to at most 2^14 (w: the largest that the row has seen, relative to its
// running maximum).  That is 22 bits of every value down to 2^-17 of the largest and, below that, 2^-38 of the largest
// in absolute terms, against the 24 bits of fp32; sums are fp32.  So a position's weight is off by no more than
// 2^-38 of what the row's largest term has, whatever the sizes of the V that other rows see or that the softmax
// ignores.  (The power of two of w by the scales b alone, which are at hand before the weights, would save the search for the
// largest, 1 % of the time with a shared prefix; but a large b that a row does not see, or that has no weight, would leave
// the others no bits.  One fp16 part would leave 11 bits: errors of 1e-4 where the fp32 outputs should have 1e-6.  bf16
// parts need three, and half as much again of the matrix instructions.)
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
//           takes time).  Every wave holds 16 rows of its own, and all walk the same tiles, which the workgroup turns
//           into fp16 once and keeps in LDS in the order of the matrix instructions' lanes.
//
// What bounds it.  64 sequences of up to 8192 positions, 8 x 128 dims: 126 us, 5.5 TB/s of codes, against the 6.4 of a
// plain read.  16 of up to 1024, 32 x 64: 13.4 us, of which the memory takes 7.  128 sequences over 8192 shared positions,
// 8 x 128 dims: 62 us; per 16 rows and 64 positions 280 vector instructions (softmax, splitting, the share of turning
// codes into fp16) beside 64 matrix instructions of 16 clocks, 2280 clocks where issue alone would take about 1710.
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
constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLeast = 7.8886090522101181e-31f;   // 2^-100: no power of two below it is used as a scale of q
constexpr float kLeastW = 1.9259299443872359e-34f;  // 2^-112: nor one below this for w (2^-39 of it is less than fp32 holds)

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
    // a - h exactly, h read as fp16 by the same instruction (written as such, the compiler converts h first)
    float ra, rb;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(h), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(h), "v"(b));
    l = half2v{(_Float16)ra, (_Float16)rb};
}

__device__ __forceinline__ void put(half8 &v, int at, half2v h) { v[at] = h[0], v[at + 1] = h[1]; }

__device__ __forceinline__ float max_groups(float v)   // over the four lanes of a column
{
    float2 p = swap32(v, v);
    v = fmaxf(p.x, p.y);
    p = swap16(v, v);
    return fmaxf(p.x, p.y);
}

__device__ __forceinline__ float sum_groups(float v)
{
    float2 p = swap32(v, v);
    v = p.x + p.y;
    p = swap16(v, v);
    return p.x + p.y;
}

// Keeps the compiler from moving instructions across: without it, it fetches all operands of a tile before
// the first product and runs out of registers, or fetches them right where they are used and waits.
__device__ __forceinline__ void here() { __builtin_amdgcn_sched_barrier(0); }

// A wave-uniform flag that the compiler takes for a new one at every use: a loop that asks for it is not copied for
// each of its values.
__device__ __forceinline__ bool asked(int flag)
{
    asm volatile("" : "+v"(flag));
    return __builtin_amdgcn_readfirstlane(flag) != 0;
}

// Orders a wave's own accesses to LDS: what some lanes write, others read.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

struct KTile {
    uint4v a[4][NC > 0 ? NC : 1];
    uint2v b[4];
};
struct VTile {
    uint4v a[ND];
};

// NT: past the caches (what a call reads once and they would not hold until the next call).
template <bool NT, typename T>
__device__ __forceinline__ T fetch(const uint8_t *p)
{
    return NT ? __builtin_nontemporal_load((const T *)p) : *(const T *)p;
}

template <bool NT>
__device__ __forceinline__ void load_k(KTile &k, const uint8_t *rec, int g, int col)
{
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const uint8_t *p = rec + (16 * t + col) * W;
#pragma unroll
        for (int n = 0; n < NC; n++) k.a[t][n] = fetch<NT, uint4v>(p + 64 * n + 16 * g);
        if constexpr (TAIL) k.b[t] = fetch<NT, uint2v>(p + 64 * NC + 8 * g);
    }
}

template <bool NT>
__device__ __forceinline__ void load_v(VTile &v, const uint8_t *rec, int g, int col)
{
    const uint8_t *p = rec + kKvTile * W + col * kKvTile + 16 * g;
#pragma unroll
    for (int n = 0; n < ND; n++) v.a[n] = fetch<NT, uint4v>(p + 16 * kKvTile * n);
}

struct RowRef {          // a row of the batch
    bool valid;
    int token, head;     // token: sequence * n_q + i
};

// id / group: the product with the rounded reciprocal is off by less than 2^-20 (id < 2^28, group < 2^16) and the half
// keeps it that far from whole numbers.
__device__ __forceinline__ int by_group(int id, double inv_group) { return (int)(((double)id + 0.5) * inv_group); }

// Sixteen rows' queries on their way from memory, read row by row, to the lanes of the second operands of K q^T.
// The 16-byte chunks of row r are permuted by r, so that 16 lanes reading one chunk of 16 rows meet few bank conflicts.
struct QRows {
    float4v c[16][W / 4];
};

// Chunks of rows, `count` threads from `first` on; rows that do not exist and dims beyond head_dim are 0.
template <typename RowOf>
__device__ __forceinline__ void bring_q(const AttnQ8Args &a, QRows &S, int first, int count, RowOf row_of)
{
    for (int i = first; i < 16 * (W / 4); i += count) {
        const int row = i / (W / 4), ch = i % (W / 4);
        const RowRef r = row_of(row);
        float4v f = {0, 0, 0, 0};
        if (r.valid && 4 * ch < a.hd) {
            const float *q = a.q + (int64_t)r.token * a.q_stride + (int64_t)r.head * a.hd + 4 * ch;
            if (a.q_vec) {
                f = *(const float4v *)q;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) f[e] = q[e];
            }
        }
        S.c[row][ch ^ (row & 7)] = f;
    }
}

// The power of two that a row of q is brought to the range of fp16 with, and the units of the products, as AttnQ8Args has
// scores.
struct QScale {
    float mul, unit;
};
// amax: the largest finite element; bad: the row holds a NaN or an infinity, and becomes NaN.
__device__ __forceinline__ QScale q_scale(const AttnQ8Args &a, float amax, bool bad)
{
    const float unit = amax > kLeast ? __uint_as_float(__float_as_uint(amax) & 0x7F800000u) : kLeast;   // 2^e
    const float mul = __uint_as_float((268u << 23) - __float_as_uint(unit));                            // 2^14 / unit
    return QScale{bad ? __uint_as_float(0x7FC00000u) : mul, unit * (1.0f / 262144.0f)};
}

// The operands of the rows in S, and the units of their products.
__device__ __forceinline__ void take_q(const AttnQ8Args &a, const QRows &S, half8 (&qh)[NK], half8 (&ql)[NK], float &xu, int g, int col)
{
    float4v f[NK][2];
    uint32_t top = 0;
#pragma unroll
    for (int n = 0; n < NK; n++) {
        // the dims of this lane's bytes: 16 g + 8 (n % 2) of piece n / 2, 8 g of the 32-wide one
        const int d = TAIL && n == NK - 1 ? 64 * NC + 8 * g : 64 * (n >> 1) + 16 * g + 8 * (n & 1);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            f[n][j] = S.c[col][(d / 4 + j) ^ (col & 7)];
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, __float_as_uint(f[n][j][e]) & 0x7FFFFFFFu);
        }
    }
    const QScale q = q_scale(a, max_groups(__uint_as_float(min(top, 0x7F7FFFFFu))), max_groups(top > 0x7F7FFFFFu ? 1.0f : 0.0f) > 0.0f);
    xu = q.unit;
#pragma unroll
    for (int n = 0; n < NK; n++)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            half2v h, l;
            split(f[n][e >> 2][e & 3] * q.mul, f[n][e >> 2][(e & 3) + 1] * q.mul, h, l);
            put(qh[n], e, h);
            put(ql[n], e, l);
        }
}

// x = K q^T of a tile; k_of(t, n): the codes of positions 16 t .. as operand n along the row.  The operands of
// the next n are made ready (LDS: requested) before the products of this one; the products of four
// position groups lie between two that add to the same sum.
template <bool LDS, typename KOf>
__device__ __forceinline__ void scores(float4v (&x)[4], const half8 (&qh)[NK], const half8 (&ql)[NK], KOf k_of)
{
    half8 k[2][4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        k[0][t] = k_of(t, 0);
        x[t] = float4v{0, 0, 0, 0};
    }
#pragma unroll
    for (int n = 0; n < NK; n++) {
        if (n + 1 < NK) {
#pragma unroll
            for (int t = 0; t < 4; t++) k[(n + 1) & 1][t] = k_of(t, n + 1);
            if (LDS) here();
        }
#pragma unroll
        for (int t = 0; t < 4; t++) x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[n & 1][t], qh[n], x[t], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < 4; t++) x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[n & 1][t], ql[n], x[t], 0, 0, 0);
        here();
    }
}

// acc += V^T w^T of a tile; v_of(n, kb): the codes of dims 16 n .. at the positions of half kb.  Two groups
// of dims at a time (ND is even), the next two made ready before their products.
template <bool LDS, typename VOf>
__device__ __forceinline__ void weigh(float4v (&acc)[ND], const half8 (&ph)[2], const half8 (&pl)[2], VOf v_of)
{
    half8 v[2][2][2];
#pragma unroll
    for (int j = 0; j < 4; j++) v[0][j >> 1][j & 1] = v_of(j >> 1, j & 1);
#pragma unroll
    for (int n0 = 0; n0 < ND; n0 += 2) {
        const int b = (n0 >> 1) & 1;
        if (n0 + 2 < ND) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[b ^ 1][j >> 1][j & 1] = v_of(n0 + 2 + (j >> 1), j & 1);
            if (LDS) here();
        }
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
#pragma unroll
            for (int n = 0; n < 2; n++)
                acc[n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b][n][kb], ph[kb], acc[n0 + n], 0, 0, 0);
#pragma unroll
            for (int n = 0; n < 2; n++)
                acc[n0 + n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[b][n][kb], pl[kb], acc[n0 + n], 0, 0, 0);
        }
        here();
    }
}

// The running softmax of a block of rows, a row per column of 16 lanes.
struct Running {
    // m: the largest x so far, that acc and l are relative to; xu: the units of x
    float m = kNegInf, l = 0.0f, xu;
    // most: the largest w so far, relative to m; unit: the power of two above it, in whose 2^-14ths acc is
    float most = 0.0f, unit = kLeastW;
    float4v acc[ND];

    __device__ __forceinline__ Running()
    {
#pragma unroll
        for (int n = 0; n < ND; n++) acc[n] = float4v{0, 0, 0, 0};
    }

    // One tile: x (K q^T) becomes the weights' parts, acc and l move to the new maximum and unit.  ks(t), vs(t): the
    // scales of this lane's positions.  With WHOLE every position counts for every row; otherwise the row sees
    // the tile's first `vis`; what is not seen weighs nothing, and sets no unit, whatever its scales hold.
    // Exponents are (x - m) c, not x c - (m c), which saves an instruction: m c rounded is off by up to 2^-24 of it, and a
    // weight that is 2^off too large leaves fp16 when scores pass 2^26.
    template <bool WHOLE, typename KsOf, typename VsOf>
    __device__ __forceinline__ void step(float4v (&x)[4], float c, KsOf ks, VsOf vs, half8 (&ph)[2], half8 (&pl)[2], int vis, int g)
    {
        float top = m;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            x[t] *= ks(t);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (!WHOLE && 16 * t + 4 * g + i >= vis) x[t][i] = kNegInf;
                top = fmaxf(top, x[t][i]);
            }
        }
        top = max_groups(top);
        // (a row that has seen nothing yet: x = -inf against 0)
        const float base = top == kNegInf ? 0.0f : top;
        const float alpha = __builtin_amdgcn_exp2f((m - base) * c);
        m = top;
        float sum = 0.0f, big = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            const float4v v = vs(t);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = __builtin_amdgcn_exp2f((x[t][i] - base) * c);
                sum += p;
                x[t][i] = p * v[i];
                if (!WHOLE && 16 * t + 4 * g + i >= vis) x[t][i] = 0.0f;
                big = fmaxf(big, x[t][i]);   // (a NaN sets no unit)
            }
        }
        l = l * alpha + sum;
        most = fmaxf(most * alpha, max_groups(big));
        const float was = alpha * unit;   // at most twice the new unit
        unit = pow2_above(fmaxf(most, kLeastW));
        const float down = was * __uint_as_float((254u << 23) - __float_as_uint(unit));   // was / unit
        if (__any(down != 1.0f)) {
#pragma unroll
            for (int n = 0; n < ND; n++) acc[n] *= down;
        }
        const float mul = __uint_as_float((268u << 23) - __float_as_uint(unit));   // 2^14 / unit
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                half2v h, r;
                split(x[t][i] * mul, x[t][i + 1] * mul, h, r);
                put(ph[t >> 1], 4 * (t & 1) + i, h);
                put(pl[t >> 1], 4 * (t & 1) + i, r);
            }
            here();
        }
    }
};

// Memory of four waves that work on one unit: first the queries, then the joining of the waves' sums.
struct Shared {
    union {
        QRows q;
        struct {
            float m[4][16], l[4][16];
            float acc[4][16][W + 4];
        };
    };
    float scale[4][2][kKvTile];   // of a wave's tile, K and V
};

// stream: the four waves take the tiles of positions [p0, p1) in turn; vis_of(row): positions that the row
// sees, counted from the slot's first, min_vis at least.
template <bool NT, typename RowOf, typename VisOf>
__device__ __forceinline__ void stream(const AttnQ8Args &a, Shared &S, const uint8_t *cache, int p0, int p1, int min_vis,
                                       RowOf row_of, VisOf vis_of)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, wave = wave_id();
    const int n_tiles = (p1 - p0 + kKvTile - 1) / kKvTile;
    constexpr size_t REC = kv_tile_bytes(W);

    const uint8_t *rec = cache + (size_t)(p0 / kKvTile + wave) * REC;
    KTile kt;
    VTile vt;
    float kone = 0.0f, vone = 0.0f;
    float (*scale)[kKvTile] = S.scale[wave];
    const auto load_scales = [&]() {
        const float *p = (const float *)(rec + 2 * kKvTile * W) + lane;
        kone = p[0], vone = p[kKvTile];
    };
    if (wave < n_tiles) {
        load_k<NT>(kt, rec, g, col);
        load_v<NT>(vt, rec, g, col);
        load_scales();
    }
    half8 qh[NK], ql[NK];
    Running R;
    bring_q(a, S.q, threadIdx.x, 256, row_of);
    __syncthreads();
    take_q(a, S.q, qh, ql, R.xu, g, col);
    const float c = a.scale_log2e * R.xu;
    const int vis = row_of(col).valid ? vis_of(col) : 0;

    // tiles that every row sees all of, then the rest: the same code with and without the bounds
    const auto go = [&](int &tile, int end, auto whole) {
        for (; tile < end; tile += 4) {
            // a position's scales per lane, to be read by the lanes whose x belongs to it
            const int at = p0 + tile * kKvTile;
            scale[0][lane] = kone;
            scale[1][lane] = vone;
            wave_fence();
            rec += 4 * REC;
            const bool more = tile + 4 < n_tiles;
            float4v x[4];
            scores<false>(x, qh, ql, [&](int t, int n) {
                if (TAIL && n == NK - 1) return halves(kt.b[t][0], kt.b[t][1]);
                return halves(kt.a[t][n >> 1][2 * (n & 1)], kt.a[t][n >> 1][2 * (n & 1) + 1]);
            });
            if (more) load_k<NT>(kt, rec, g, col);
            half8 ph[2], pl[2];
            R.template step<decltype(whole)::value>(
                x, c, [&](int t) { return *(const float4v *)&scale[0][16 * t + 4 * g]; },
                [&](int t) { return *(const float4v *)&scale[1][16 * t + 4 * g]; }, ph, pl, vis - at, g);
            weigh<false>(R.acc, ph, pl, [&](int n, int kb) { return halves(vt.a[n][2 * kb], vt.a[n][2 * kb + 1]); });
            if (more) {
                load_v<NT>(vt, rec, g, col);
                load_scales();
            }
            wave_fence();
        }
    };
    int tile = wave;
    go(tile, min(n_tiles, (min_vis - p0) / kKvTile), std::true_type{});
    go(tile, n_tiles, std::false_type{});

    __syncthreads();   // (the queries have been read)
    const float sum = sum_groups(R.l), up = R.unit * (1.0f / 16384.0f);
    if (g == 0) {
        S.m[wave][col] = R.m * R.xu;
        S.l[wave][col] = sum;
    }
#pragma unroll
    for (int n = 0; n < ND; n++) *(float4v *)&S.acc[wave][col][16 * n + 4 * g] = R.acc[n] * up;
    __syncthreads();
}

// Joins the waves' sums and writes the rows: the outputs, or with more parts to come the part's
// maximum, sum and weighted sums.
template <typename RowOf>
__device__ __forceinline__ void finish(const AttnQ8Args &a, Shared &S, int part, RowOf row_of)
{
    for (int i = threadIdx.x; i < 16 * (W / 4); i += 256) {
        const int row = i / (W / 4), d = 4 * (i % (W / 4));
        const RowRef r = row_of(row);
        if (!r.valid || d >= a.hd) continue;
        float top = kNegInf, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) top = fmaxf(top, S.m[w][row]);
        float4v o = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            // a wave without a visible position has the sum 0 (and one that saw NaN a NaN)
            const float f = S.m[w][row] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f((S.m[w][row] - top) * a.scale_log2e);
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

// A wave's share of a tile that the workgroup brings from memory to LDS: K of positions 16 wave .. and V of dims
// 16 (wave + 4 j) .., requested one tile ahead.
struct Share {
    static constexpr int NV = (ND + 3) / 4;
    uint4v ka[NC > 0 ? NC : 1], va[NV];
    uint2v kb;
    float scale;

    __device__ __forceinline__ void load(const uint8_t *rec, int wave, int g, int col)
    {
        const uint8_t *k = rec + (16 * wave + col) * W, *v = rec + kKvTile * W + col * kKvTile + 16 * g;
#pragma unroll
        for (int n = 0; n < NC; n++) ka[n] = *(const uint4v *)(k + 64 * n + 16 * g);
        if constexpr (TAIL) kb = *(const uint2v *)(k + 64 * NC + 8 * g);
#pragma unroll
        for (int j = 0; j < NV; j++)
            if (wave + 4 * j < ND) va[j] = *(const uint4v *)(v + 16 * kKvTile * (wave + 4 * j));
        if (threadIdx.x < 2 * kKvTile) scale = ((const float *)(rec + 2 * kKvTile * W))[threadIdx.x];
    }

    __device__ __forceinline__ void put_scales(float (&to)[2][kKvTile]) const
    {
        if (threadIdx.x < 2 * kKvTile) to[threadIdx.x / kKvTile][threadIdx.x % kKvTile] = scale;
    }
};

// rows: fragments of 1 KB, a lane's 16 bytes after another's: K by (t, n), V by (n, kb).
constexpr int NB = W <= 128 ? 2 : 1;   // a second buffer takes the next tile while this one is read, where there is room
struct Tiles {
    half8 k[NB][4][NK][64], v[NB][ND][2][64];
    float scale[NB][2][kKvTile];
};

// Positions [p0, p1), all seen by every row; each of the four waves has its own rows row_of(0 .. 15).  Writes the
// rows' part.
template <typename RowOf>
__device__ __forceinline__ void rows(const AttnQ8Args &a, Tiles &S, QRows *Q, const uint8_t *cache, int p0, int p1, int part,
                                     RowOf row_of)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, wave = wave_id();
    const int n_tiles = (p1 - p0 + kKvTile - 1) / kKvTile;
    constexpr size_t REC = kv_tile_bytes(W);
    const uint8_t *rec = cache + (size_t)(p0 / kKvTile) * REC;
    Share in;
    in.load(rec, wave, g, col);

    half8 qh[NK], ql[NK];
    Running R;
    bring_q(a, Q[wave], lane, 64, row_of);
    __syncthreads();
    take_q(a, Q[wave], qh, ql, R.xu, g, col);
    const float c = a.scale_log2e * R.xu;
    __syncthreads();
    const int busy = __any(row_of(0).valid);   // (a wave without rows brings its share of the tiles)

    const auto go = [&](int &tile, int end, auto whole) {
        for (; tile < end; tile++) {
            const int b = NB == 2 ? tile & 1 : 0;
            if (NB == 1 && tile > 0) __syncthreads();   // the tile before has been read
#pragma unroll
            for (int n = 0; n < NC; n++) {
                S.k[b][wave][2 * n][lane] = halves(in.ka[n][0], in.ka[n][1]);
                S.k[b][wave][2 * n + 1][lane] = halves(in.ka[n][2], in.ka[n][3]);
            }
            if constexpr (TAIL) S.k[b][wave][NK - 1][lane] = halves(in.kb[0], in.kb[1]);
#pragma unroll
            for (int j = 0; j < Share::NV; j++)
                if (wave + 4 * j < ND) {
                    S.v[b][wave + 4 * j][0][lane] = halves(in.va[j][0], in.va[j][1]);
                    S.v[b][wave + 4 * j][1][lane] = halves(in.va[j][2], in.va[j][3]);
                }
            in.put_scales(S.scale[b]);
            rec += REC;
            if (tile + 1 < n_tiles) in.load(rec, wave, g, col);
            __syncthreads();
            if (!asked(busy)) continue;
            float4v x[4];
            scores<true>(x, qh, ql, [&](int t, int n) { return S.k[b][t][n][lane]; });
            half8 ph[2], pl[2];
            R.template step<decltype(whole)::value>(
                x, c, [&](int t) { return *(const float4v *)&S.scale[b][0][16 * t + 4 * g]; },
                [&](int t) { return *(const float4v *)&S.scale[b][1][16 * t + 4 * g]; }, ph, pl, p1 - p0 - tile * kKvTile, g);
            weigh<true>(R.acc, ph, pl, [&](int n, int kb) { return S.v[b][n][kb][lane]; });
        }
    };
    int tile = 0;
    go(tile, (p1 - p0) / kKvTile, std::true_type{});
    go(tile, n_tiles, std::false_type{});
    const RowRef r = row_of(col);
    const float sum = sum_groups(R.l), up = R.unit * (1.0f / 16384.0f);
    if (!r.valid) return;
    const int64_t id = (int64_t)part * a.n_rows + (int64_t)r.token * a.n_head + r.head;
    if (g == 0) a.part_ml[id * 2] = R.m * R.xu, a.part_ml[id * 2 + 1] = sum;
    float *dst = a.part_acc + id * a.hd + 4 * g;
#pragma unroll
    for (int n = 0; n < ND; n++)
        if (16 * n + 4 * g < a.hd) *(float4v *)(dst + 16 * n) = R.acc[n] * up;
}

// PRE: how the prefix is gone through; the sequences' own positions: stream, NT or not.
template <AttnQ8Pre PRE, bool NT>
__global__ __launch_bounds__(256, W <= 64 ? 3 : W <= 128 ? 2 : 1) void k_attn_q8(const AttnQ8Args a)
{
    union Mem {
        Shared own;
        std::conditional_t<PRE == PRE_ROWS, Tiles, int> tiles;
        QRows q[PRE == PRE_ROWS ? 4 : 1];
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
        const int row0 = PRE == PRE_ROWS ? (rb * 4 + wave_id()) * 16 : rb * 16, n_rows = a.n_seq * a.n_q * group;
        const auto row_of = [&](int r) {
            const int id = row0 + r;
            const int t = by_group(id, a.inv_group);
            return RowRef{id < n_rows, t, head * group + id - t * group};
        };
        const uint8_t *cache = a.cache + (size_t)(a.prefix_slot * (int64_t)a.n_kv + head) * a.head_bytes;
        if constexpr (PRE == PRE_ROWS) {
            rows(a, S.tiles, S.q, cache, p0, p1, split, row_of);
        } else {
            stream<false>(a, S.own, cache, p0, p1, a.prefix_len, row_of, [&](int) { return a.prefix_len; });
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
        const int t = by_group(id, a.inv_group);
        return RowRef{id < n_rows, seq * a.n_q + t, head * group + id - t * group};
    };
    const int part = a.pre_splits + split;
    if (p0 < p1) {
        // the first of the n_q tokens sees len - n_q + 1 positions, each further one sees one more
        stream<NT>(a, S.own, a.cache + (size_t)(slot * (int64_t)a.n_kv + head) * a.head_bytes, p0, p1, len - a.n_q + 1,
                   row_of, [&](int r) { return len - a.n_q + 1 + by_group(row0 + r, a.inv_group); });
        finish(a, S.own, part, row_of);
        return;
    }
    // nothing here: zeros, or a part without weight
    for (int i = threadIdx.x; i < 16 * W; i += 256) {
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
}

}  // namespace

#define SMX_LAUNCH_NAME_(w) launch_attn_q8_w##w
#define SMX_LAUNCH_NAME(w) SMX_LAUNCH_NAME_(w)
hipError_t SMX_LAUNCH_NAME(SMX_ATTN_W)(const AttnQ8Args &a, const AttnQ8Plan &p, hipStream_t s)
{
    const unsigned blocks = (unsigned)p.blocks;
    if (p.pre == PRE_NONE && p.past_caches) k_attn_q8<PRE_NONE, true><<<blocks, 256, 0, s>>>(a);
    else if (p.pre == PRE_NONE) k_attn_q8<PRE_NONE, false><<<blocks, 256, 0, s>>>(a);
    else if (p.pre == PRE_STREAM) k_attn_q8<PRE_STREAM, false><<<blocks, 256, 0, s>>>(a);
    else k_attn_q8<PRE_ROWS, false><<<blocks, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
