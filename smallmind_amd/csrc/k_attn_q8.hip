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
// need two lane exchanges.  The contraction order of q K^T is whatever 16-byte loads give.  Nothing
// passes through LDS until the four waves of a workgroup, which take tiles in turn, join their sums.
// The positions are cut into chunks, a workgroup each (and for the shared prefix the rows into
// blocks of 16 or 32); k_attn_q8_join adds up what the chunks found.  K of the next tile is loaded as
// soon as this tile's products have used it, V likewise.
#include "smx_device.h"
#include "smx_internal.h"
#include "smx_attn_q8.h"

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

// MT blocks of 16 rows of one KV head against positions [p0, p1) of one slot.  vis_of(row): positions that
// the row sees, counted from the slot's first.  Results of the workgroup: rows' maxima and sums, and the
// weighted sums of V in S.
template <int MT>
struct Shared {
    float m[4][16 * MT], l[4][16 * MT];
    float acc[4][16 * MT][W + 4];
};

struct RowRef {          // a row of the batch
    bool valid;
    int token, head;     // token: sequence * n_q + i
};

template <int MT, typename RowOf, typename VisOf>
__device__ __forceinline__ void attend(const AttnQ8Args &a, Shared<MT> &S, const uint8_t *cache, int p0, int p1, int min_vis,
                                       RowOf row_of, VisOf vis_of)
{
    const int lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15, wave = wave_id();
    const int n_tiles = (p1 - p0 + kKvTile - 1) / kKvTile;
    constexpr size_t REC = kv_tile_bytes(W);

    half8 qh[MT][NK], ql[MT][NK];
    float c[MT];
    int vis[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const RowRef r = row_of(16 * mt + col);
        vis[mt] = r.valid ? vis_of(16 * mt + col) : 0;
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
        const float mul = bad ? __uint_as_float(0x7FC00000u) : 16384.0f / unit;
        c[mt] = a.scale_log2e * (unit * (1.0f / 16384.0f));
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = bad ? mul : f[n][e] * mul;
                const _Float16 h = (_Float16)x;
                qh[mt][n][e] = h;
                ql[mt][n][e] = (_Float16)(x - (float)h);
            }
    }

    float4v acc[MT][ND];
    // m: the largest x so far; mc: c m as rounded, the exponent that acc and l are relative to
    float m[MT], mc[MT], l[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        m[mt] = mc[mt] = kNegInf;
        l[mt] = 0.0f;
#pragma unroll
        for (int n = 0; n < ND; n++) acc[mt][n] = float4v{0, 0, 0, 0};
    }
    float vref = kLeast;   // power of two, at least every V scale so far

    const uint8_t *rec = cache + (size_t)(p0 / kKvTile + wave) * REC;
    KTile kt;
    VTile vt;
    if (wave < n_tiles) {
        load_k(kt, rec, g, col);
        load_v(vt, rec, g, col);
    }
    for (int tile = wave; tile < n_tiles; tile += 4) {
        const float *scales = (const float *)(rec + 2 * kKvTile * W);
        float4v ks[4], vs[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            ks[t] = *(const float4v *)(scales + 16 * t + 4 * g);
            vs[t] = *(const float4v *)(scales + kKvTile + 16 * t + 4 * g);
        }
        const uint8_t *next = rec + 4 * REC;
        const bool more = tile + 4 < n_tiles;

        float4v x[MT][4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++) x[mt][t] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int n = 0; n < NK; n++) {
                half8 kk;
                if (TAIL && n == NK - 1) kk = halves(kt.b[t][0], kt.b[t][1]);
                else kk = halves(kt.a[t][n >> 1][2 * (n & 1)], kt.a[t][n >> 1][2 * (n & 1) + 1]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    x[mt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, qh[mt][n], x[mt][t], 0, 0, 0);
                    x[mt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, ql[mt][n], x[mt][t], 0, 0, 0);
                }
            }
        }
        if (more) load_k(kt, next, g, col);

        // x times the K scales; what a row does not see is -inf, and weighs nothing whatever its V scale holds
        const int at = p0 + tile * kKvTile;
        const bool whole = at + kKvTile <= min_vis;
        const int left = p1 - at;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int p = 16 * t + 4 * g + i;
                if (!whole && p >= left) vs[t][i] = 0.0f;
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    float f = x[mt][t][i] * ks[t][i];
                    if (!whole && at + p >= vis[mt]) f = kNegInf;
                    x[mt][t][i] = f;
                }
            }
        // the V scales relative to a power of two that grows with them
        float vmax = 0.0f;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) vmax = fmaxf(vmax, vs[t][i]);
        vmax = max_groups(vmax);
        const float vnew = fmaxf(vref, pow2_above(fmaxf(vmax, kLeast)));
        const float vmul = __uint_as_float((268u << 23) - __float_as_uint(vnew));   // 2^14 / vnew
        const float vdown = vref * (vmul * (1.0f / 16384.0f));
        vref = vnew;
#pragma unroll
        for (int t = 0; t < 4; t++) vs[t] *= vmul;

        half8 ph[MT][2], pl[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float top = m[mt];
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, x[mt][t][i]);
            top = max_groups(top);
            // (a row that has seen nothing yet: x = -inf against 0)
            const float now = top == kNegInf ? 0.0f : top * c[mt];
            const float alpha = __builtin_amdgcn_exp2f(mc[mt] - now);
            if (top != kNegInf) m[mt] = top, mc[mt] = now;
            float sum = 0.0f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[mt][t][i], c[mt], -now));
                    sum += p;
                    float w = p * vs[t][i];
                    if (!whole && at + 16 * t + 4 * g + i >= vis[mt]) w = 0.0f;
                    const _Float16 h = (_Float16)w;
                    ph[mt][t >> 1][4 * (t & 1) + i] = h;
                    pl[mt][t >> 1][4 * (t & 1) + i] = (_Float16)(w - (float)h);
                }
            l[mt] = l[mt] * alpha + sum;
            const float down = alpha * vdown;
            if (__any(down != 1.0f)) {
#pragma unroll
                for (int n = 0; n < ND; n++) acc[mt][n] *= down;
            }
        }
#pragma unroll
        for (int n = 0; n < ND; n++)
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const half8 vv = halves(vt.a[n][2 * kb], vt.a[n][2 * kb + 1]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    acc[mt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, ph[mt][kb], acc[mt][n], 0, 0, 0);
                    acc[mt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, pl[mt][kb], acc[mt][n], 0, 0, 0);
                }
            }
        if (more) load_v(vt, next, g, col);
        rec = next;
    }

    // the waves' sums, each in units of its own maximum (in powers of two) and V scale
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const int row = 16 * mt + col;
        const float sum = sum_groups(l[mt]), up = vref * (1.0f / 16384.0f);
        if (g == 0) {
            S.m[wave][row] = mc[mt];
            S.l[wave][row] = sum;
        }
#pragma unroll
        for (int n = 0; n < ND; n++) *(float4v *)&S.acc[wave][row][16 * n + 4 * g] = acc[mt][n] * up;
    }
    __syncthreads();
}

// Joins the four waves' sums and writes the rows: the outputs, or with more parts to come the part's
// maximum (in powers of two), sum and weighted sums.
template <int MT, typename RowOf>
__device__ __forceinline__ void finish(const AttnQ8Args &a, Shared<MT> &S, int part, RowOf row_of)
{
    for (int i = threadIdx.x; i < 16 * MT * (W / 4); i += 256) {
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
            const float f = S.m[w][row] == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(S.m[w][row] - top);
            if (S.l[w][row] == 0.0f) continue;
            sum += S.l[w][row] * f;
            o += *(const float4v *)&S.acc[w][row][d] * f;
        }
        const int64_t id = (int64_t)r.token * a.n_head + r.head;
        if (a.direct) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            float *dst = a.out + id * a.hd + d;
#pragma unroll
            for (int e = 0; e < 4; e++) dst[e] = o[e] * inv;
        } else {
            float *ml = a.part_ml + (part * a.n_rows + id) * 2;
            if (d == 0) ml[0] = top, ml[1] = sum;
            float *dst = a.part_acc + (part * a.n_rows + id) * a.hd + d;
#pragma unroll
            for (int e = 0; e < 4; e++) dst[e] = o[e];
        }
    }
}

// MTO, MTP: 16-row blocks per wave over the sequences' own positions and over the prefix.
template <int MTO, int MTP>
__global__ __launch_bounds__(256) void k_attn_q8(const AttnQ8Args a)
{
    constexpr int MTM = MTO > MTP ? MTO : MTP;
    __shared__ Shared<MTM> S;
    const int group = a.n_head / a.n_kv;
    int b = blockIdx.x;
    if (b < a.pre_wgs) {
        // (chunk, KV head) fastest: workgroups that read the same positions are a multiple of 8 apart
        const int pairs = a.n_kv * a.pre_splits, pair = b % pairs, rb = b / pairs;
        const int head = pair % a.n_kv, split = pair / a.n_kv;
        const int p0 = split * a.pre_chunk, p1 = min(a.prefix_len, p0 + a.pre_chunk);
        const int row0 = rb * 16 * MTP, n_rows = a.n_seq * a.n_q * group;
        const auto row_of = [&](int r) {
            const int id = row0 + r;
            return RowRef{id < n_rows, id / group, head * group + id % group};
        };
        Shared<MTP> &T = *(Shared<MTP> *)&S;
        attend<MTP>(a, T, a.cache + (size_t)(a.prefix_slot * (int64_t)a.n_kv + head) * a.head_bytes, p0, p1, a.prefix_len,
                    row_of, [&](int) { return a.prefix_len; });
        finish<MTP>(a, T, split, row_of);
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
    const int row0 = rb * 16 * MTO, n_rows = a.n_q * group;
    const auto row_of = [&](int r) {
        const int id = row0 + r;
        return RowRef{id < n_rows, seq * a.n_q + id / group, head * group + id % group};
    };
    const int part = a.pre_splits + split;
    Shared<MTO> &T = *(Shared<MTO> *)&S;
    if (p0 >= p1) {
        // nothing here: zeros, or a part without weight
        for (int i = threadIdx.x; i < 16 * MTO * W; i += 256) {
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
    attend<MTO>(a, T, a.cache + (size_t)(slot * (int64_t)a.n_kv + head) * a.head_bytes, p0, p1, len - a.n_q + 1, row_of,
                [&](int r) { return len - a.n_q + 1 + (row0 + r) / group; });
    finish<MTO>(a, T, part, row_of);
}

}  // namespace

#define SMX_LAUNCH_NAME_(w) launch_attn_q8_w##w
#define SMX_LAUNCH_NAME(w) SMX_LAUNCH_NAME_(w)
hipError_t SMX_LAUNCH_NAME(SMX_ATTN_W)(const AttnQ8Args &a, int mt_own, int mt_pre, unsigned blocks, hipStream_t s)
{
    if (mt_own == 1 && mt_pre == 1) {
        k_attn_q8<1, 1><<<blocks, 256, 0, s>>>(a);
    } else if constexpr (kAttnQ8TwoBlocks<SMX_ATTN_W>) {
        if (mt_own == 1) k_attn_q8<1, 2><<<blocks, 256, 0, s>>>(a);
        else k_attn_q8<2, 2><<<blocks, 256, 0, s>>>(a);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace smx
