// k_attn_mass.hip -- the attention weight that every position of the paged KV cache receives from a batch's new tokens,
// summed over them and the query heads of a KV head, added to what it has received.  Built once per row width
// and element type.
//
// Mathematics.  out[p] = mass[p] + sum over rows of 2^(s(row, p) - lse(row)), with the scores of the attention and the logarithm of
// its sums, fp32.  Every output has one thread, or one per part of the rows, whose sums are added in their order.
//
// Layout.  Scores as in k_attn_paged.hip, S^T = K q^T, a row per column of lanes, which are added at the end.
//   few rows (up to 32 per KV head): a wave keeps their queries as operands in registers and takes 32 positions in turn, K on its
//     way from memory one turn ahead.
//   many rows: a wave keeps the K of 32 or 64 positions as operands in registers and goes through the rows, 32 at a time, whose operands the
//     workgroup's four waves lay out in LDS for one another, the next ones' on their way in the meantime.
#include "smx_attn_paged_dev.h"

namespace smx {

namespace {

constexpr int kWaves = 4;
constexpr int KT = W <= 128 ? 2 : 1;      // 32-position groups of a wave (many rows)
constexpr int kKeys = 32 * KT * kWaves;   // positions of a workgroup

// The sum over a row of lanes' first n columns (at least; the others hold 0).
__device__ __forceinline__ float sum_columns(float v, int n)
{
    if (n > 1) v += dpp_mov<0xB1>(v);
    if (n > 2) v += dpp_mov<0x4E>(v);
    if (n > 4) v += dpp_mov<0x141>(v);
    if (n > 8) v += dpp_mov<0x140>(v);
    if (n > 16) v += swap16_other(v);
    return v;
}

// What the positions of 32 from `at` on have received, in the first lane of each half.
__device__ __forceinline__ void give(const AttnPgArgs &a, const Seq &s, int pair, int part, int at, int h, const float16v &sum)
{
    const int64_t row = (int64_t)pair * a.max_len, pairs = (int64_t)a.n_seq * a.c.n_kv;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int p = at + pos32(i, h);
        if (p >= a.max_len) continue;
        if (a.mass_parts > 1) {
            a.mass_part[part * pairs * a.max_len + row + p] = sum[i];
            continue;
        }
        const float was = a.mass && p < a.mass_width ? a.mass[pair * a.mass_stride + p] : 0.0f;
        a.mass_out[row + p] = p < s.len ? was + sum[i] : 0.0f;
    }
}

// K of 32 positions from `at` on as operands.
__device__ __forceinline__ void load_k(const AttnPgArgs &a, const Seq &s, Pages &P, int at, int lane, elem8 (&k)[NK], bool &there0, bool &there1)
{
    P.go(a, s, at / kPgGroup);
    const Rows16 r0 = P.rows(a, at / kPgGroup), r1 = P.rows(a, at / kPgGroup + 1);
    const uint8_t *p = (lane & 16 ? r1.p : r0.p) + (lane & 15) * ROW;
#pragma unroll
    for (int n = 0; n < NK; n++) k[n] = *(const elem8 *)(p + 16 * pg_unit(W, 2 * n + (lane >> 5), lane & 15));
    there0 = r0.there, there1 = r1.there;
}

// What a row's products become a weight with: the shape of its scores, and lse as an exponent of 2.
__device__ __forceinline__ float lse_of(const AttnPgArgs &a, const Row &r)
{
    const float l = a.lse_in[(int64_t)r.token * a.n_head + r.head];
    // (a row that sees nothing has -inf; one past the last repeats that one and counts for nothing)
    return !r.valid ? __builtin_huge_valf() : l == -__builtin_huge_valf() ? 0.0f : l * 1.4426950408889634f;
}

// ---- few rows ----------------------------------------------------------------------------------------
// A workgroup takes a share of a sequence's positions, 32 at a time in turn with its other waves.
template <bool F32>
__global__ __launch_bounds__(kWaves * 64) void k_attn_mass_few(const AttnPgArgs a)
{
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const int pairs = a.n_seq * a.c.n_kv, pair = blockIdx.x % pairs, share = blockIdx.x / pairs;
    const int b = pair / a.c.n_kv, head = pair - b * a.c.n_kv;
    const Seq s = seq_of(a, b);
    const int step = 32 * kWaves * (gridDim.x / pairs);
    int at = 32 * (kWaves * share + wave);
    elem8 k[2][NK];
    bool there[2][2];
    const bool any = s.rows > 0 && at < s.len;
    if (any) {
        Pages P(a, s, head, at / kPgGroup);
        load_k(a, s, P, at, lane, k[0], there[0][0], there[0][1]);
        const Row r = row_of(a, s, head, lane & 31);
        const float lse = lse_of(a, r);
        Query<F32> Q;
        load_q<F32>(a, r, h, Q);
        const Shape S(a, r, Q.unit);
        const Bounds B = bounds_of(a, s, s.first, row_of(a, s, head, s.rows - 1).t);
        const auto go = [&](const elem8 (&kk)[NK], bool th0, bool th1, elem8 (&next)[NK], bool (&th)[2]) {
            if (at + step < s.len) load_k(a, s, P, at + step, lane, next, th[0], th[1]);
            float16v x;
            if (B.none(s.pre, at, 32)) {
                x = float16v(0.0f);
            } else {
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int q = 0; q < kParts<F32>; q++) x = mfma(kk[n], Q.q[q][n], n || q ? x : float16v(0.0f));
                if (S.shaped) shape<true>(a, S, x, r.t, at, h);   // (the sums are fp32 whatever the queries)
                if (!th0 || !th1 || !B.whole(s.pre, at, 32)) mask(x, seen(a, s, r.t, at, h, th0, th1));
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] = sum_columns(__builtin_amdgcn_exp2f(__builtin_fmaf(x[i], S.c, -lse)), s.rows);
            }
            if ((lane & 31) == 0) give(a, s, pair, 0, at, h, x);
            at += step;
        };
        while (at < s.len) {
            go(k[0], there[0][0], there[0][1], k[1], there[1]);
            if (at < s.len) go(k[1], there[1][0], there[1][1], k[0], there[0]);
        }
    }
    // positions that nobody sees: what they had, 0 beyond the sequence
    for (; at < a.max_len; at += step)
        if ((lane & 31) == 0) give(a, s, pair, 0, at, h, float16v(0.0f));
}

// ---- many rows ---------------------------------------------------------------------------------------
// Row blocks laid out at a time.
template <bool F32> constexpr int kBlocks = kParts<F32> * W <= 256 ? 4 : kParts<F32> * W <= 512 ? 2 : 1;

template <bool F32> struct Stage {
    elem8 q[kBlocks<F32>][kParts<F32>][NK][64];
    float in[kBlocks<F32>][32], slope[kBlocks<F32>][32], lse[kBlocks<F32>][32];
    int t[kBlocks<F32>][32];
};

template <bool F32>
__global__ __launch_bounds__(kWaves * 64) void k_attn_mass(const AttnPgArgs a)
{
    constexpr int NB = kBlocks<F32>, NP = kParts<F32>;
    __shared__ Stage<F32> M;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const int pairs = a.n_seq * a.c.n_kv, pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int tiles = (a.max_len + kKeys - 1) / kKeys, tile = rest % tiles, part = rest / tiles;
    const int b = pair / a.c.n_kv, head = pair - b * a.c.n_kv;
    const Seq s = seq_of(a, b);
    const int k0 = tile * kKeys, at = k0 + 32 * KT * wave;
    // the tokens that may see one of these positions
    int t_lo = 0, t_hi = s.rows / a.group;
    if (k0 >= s.pre) {
        t_lo = max(0, k0 - s.first);
        if (a.window > 0) t_hi = (int)min((int64_t)t_hi, max((int64_t)0, (int64_t)k0 + kKeys - 1 + a.window - s.first));
    }
    const int first = t_lo * a.group, blocks = k0 < s.len ? max(0, (t_hi * a.group - first + 32 * NB - 1) / (32 * NB)) : 0;
    const int per = (blocks + a.mass_parts - 1) / a.mass_parts, s0 = part * per, s1 = min(blocks, s0 + per);
    float16v sum[KT];
#pragma unroll
    for (int t = 0; t < KT; t++) sum[t] = float16v(0.0f);
    if (s0 < s1) {
        Pages P(a, s, head, at / kPgGroup);
        elem8 k[KT][NK];
        bool there[KT][2], all = true;
#pragma unroll
        for (int t = 0; t < KT; t++) {
            load_k(a, s, P, at + 32 * t, lane, k[t], there[t][0], there[t][1]);
            all = all && there[t][0] && there[t][1];
        }
        Query<F32> Q;
        float lse = 0.0f;
        Row r{};
        const auto fetch = [&](int st) {
            r = row_of(a, s, head, first + (st * NB + wave) * 32 + (lane & 31));
            load_q<F32>(a, r, h, Q);
            lse = lse_of(a, r);
        };
        if (wave < NB) fetch(s0);
        for (int st = s0; st < s1; st++) {
            __syncthreads();   // the rows before have been read
            if (wave < NB) {
#pragma unroll
                for (int q = 0; q < NP; q++)
#pragma unroll
                    for (int n = 0; n < NK; n++) M.q[wave][q][n][lane] = Q.q[q][n];
                if (h == 0) {
                    const Shape S(a, r, Q.unit);
                    M.in[wave][lane] = S.in, M.slope[wave][lane] = S.slope, M.lse[wave][lane] = lse, M.t[wave][lane] = r.t;
                }
            }
            __syncthreads();
            if (wave < NB && st + 1 < s1) fetch(st + 1);
            const int row0 = first + st * 32 * NB;
            for (int j = 0; j < NB; j++) {
                if (row0 + 32 * j >= s.rows) break;
                const int c = lane & 31, t = M.t[j][c];
                const Bounds B = bounds_of(a, s, t, __builtin_amdgcn_readlane(t, 31));
                if (at >= s.len || B.none(s.pre, at, 32 * KT)) continue;
                Shape S;
                S.shaped = a.cap_in != 0.0f || a.slopes;
                S.in = M.in[j][c], S.slope = M.slope[j][c], S.c = S.shaped ? 1.0f : S.in;
                const float l = M.lse[j][c];
                float16v x[KT];
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int q = 0; q < NP; q++) {
                        const elem8 qq = M.q[j][q][n][lane];
#pragma unroll
                        for (int u = 0; u < KT; u++) x[u] = mfma(k[u][n], qq, n || q ? x[u] : float16v(0.0f));
                    }
                if (S.shaped) {
#pragma unroll
                    for (int u = 0; u < KT; u++) shape<true>(a, S, x[u], t, at + 32 * u, h);   // (the sums are fp32 whatever the queries)
                }
                if (!all || !B.whole(s.pre, at, 32 * KT)) {
#pragma unroll
                    for (int u = 0; u < KT; u++) mask(x[u], seen(a, s, t, at + 32 * u, h, there[u][0], there[u][1]));
                }
#pragma unroll
                for (int u = 0; u < KT; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[u][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], S.c, -l));
            }
        }
    }
#pragma unroll
    for (int u = 0; u < KT; u++) {
#pragma unroll
        for (int i = 0; i < 16; i++) sum[u][i] = sum_columns(sum[u][i], 32);
        if ((lane & 31) == 0) give(a, s, pair, part, at + 32 * u, h, sum[u]);
    }
}

}  // namespace

#define SMX_PG_NAME_(f, w, b) f##_w##w##_b##b
#define SMX_PG_NAME(f, w, b) SMX_PG_NAME_(f, w, b)
hipError_t SMX_PG_NAME(launch_attn_mass, SMX_PG_W, SMX_PG_BF16)(const AttnPgArgs &a, const MassPgPlan &p, hipStream_t s)
{
    const unsigned n = (unsigned)p.blocks;
    if (p.few && a.io == PG_F32) k_attn_mass_few<true><<<n, kWaves * 64, 0, s>>>(a);
    else if (p.few) k_attn_mass_few<false><<<n, kWaves * 64, 0, s>>>(a);
    else if (a.io == PG_F32) k_attn_mass<true><<<n, kWaves * 64, 0, s>>>(a);
    else k_attn_mass<false><<<n, kWaves * 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
