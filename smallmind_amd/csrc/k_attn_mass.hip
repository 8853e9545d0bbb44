// k_attn_mass.hip -- the attention weight that every position of the paged KV cache receives from a batch's new tokens,
// summed over them and the query heads of a KV head, added to what it has received.  Built once per row width
// and element type.
//
// Mathematics.  out[p] = mass[p] + sum over rows of 2^(s(row, p) - lse(row)), with the scores of the attention and the logarithm of
// its sums, fp32.  Every output has one thread, or one per part of the rows, whose sums are added in their order.
//
// Layout.  Scores as in k_attn_paged.hip, S^T = K q^T, but here a wave keeps 32 positions' K as operands in registers and
// goes through the rows, 32 at a time, whose operands the workgroup's four waves lay out in LDS for one another.  A lane
// keeps 16 positions' sums over its own columns; the columns are added at the end.
#include "smx_attn_paged_dev.h"

namespace smx {

namespace {

constexpr int kWaves = 4;
constexpr int kKeys = 32 * kWaves;     // positions of a workgroup

// Row blocks laid out at a time.
template <bool F32> constexpr int kBlocks = kParts<F32> * W <= 256 ? 4 : kParts<F32> * W <= 512 ? 2 : 1;

template <bool F32> struct Stage {
    elem8 q[kBlocks<F32>][kParts<F32>][NK][64];
    float unit[kBlocks<F32>][64], lse[kBlocks<F32>][64];
};

template <bool F32>
__global__ __launch_bounds__(kWaves * 64) void k_attn_mass(const AttnPgArgs a)
{
    constexpr int NB = kBlocks<F32>;
    __shared__ Stage<F32> M;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const int pairs = a.n_seq * a.c.n_kv, pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int tiles = (a.max_len + kKeys - 1) / kKeys, tile = rest % tiles, part = rest / tiles;
    const int b = pair / a.c.n_kv, head = pair - b * a.c.n_kv;
    const Seq s = seq_of(a, b);
    const int k0 = tile * kKeys, at = k0 + 32 * wave;
    // the tokens that may see one of these positions
    int t_lo = 0, t_hi = s.rows / a.group;
    if (k0 >= s.pre) {
        t_lo = max(0, k0 - s.first);
        if (a.window > 0) t_hi = min((int64_t)t_hi, max((int64_t)0, (int64_t)k0 + kKeys - 1 + a.window - s.first));
    }
    const int first = t_lo * a.group, blocks = k0 < s.len ? max(0, (t_hi * a.group - first + 32 * NB - 1) / (32 * NB)) : 0;
    const int per = (blocks + a.mass_parts - 1) / a.mass_parts, s0 = part * per, s1 = min(blocks, s0 + per);
    float16v sum;
#pragma unroll
    for (int i = 0; i < 16; i++) sum[i] = 0.0f;
    if (s0 < s1) {
        const Pages P(a, s, head, at / kPgGroup);
        const Rows16 r0 = P.rows(a, at / kPgGroup), r1 = P.rows(a, at / kPgGroup + 1);
        const uint8_t *p = (lane & 16 ? r1.p : r0.p) + (lane & 15) * ROW;
        elem8 k[NK];
#pragma unroll
        for (int n = 0; n < NK; n++) k[n] = *(const elem8 *)(p + 16 * pg_unit(W, 2 * n + h, lane & 15));
        for (int st = s0; st < s1; st++) {
            const int row0 = first + st * 32 * NB;
            __syncthreads();   // the rows before have been read
            if (wave < NB) {
                Query<F32> Q;
                const Row r = row_of(a, s, head, row0 + 32 * wave + (lane & 31));
                load_q<F32>(a, r, h, Q);
#pragma unroll
                for (int q = 0; q < kParts<F32>; q++)
#pragma unroll
                    for (int n = 0; n < NK; n++) M.q[wave][q][n][lane] = Q.q[q][n];
                M.unit[wave][lane] = Q.unit;
                const float lse = a.lse_in[(int64_t)r.token * a.n_head + r.head];
                M.lse[wave][lane] = lse == -__builtin_huge_valf() ? 0.0f : lse * 1.4426950408889634f;   // (it sees nothing)
            }
            __syncthreads();
            for (int j = 0; j < NB; j++) {
                const int id0 = row0 + 32 * j;
                if (id0 >= s.rows) break;
                const Bounds B = bounds_of(a, s, id0, 32);
                if (at >= s.len || B.none(s.pre, at, 32)) continue;
                const Row r = row_of(a, s, head, id0 + (lane & 31));
                const Shape S(a, r, M.unit[j][lane]);
                float16v x;
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] = 0.0f;
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int q = 0; q < kParts<F32>; q++) x = mfma(k[n], M.q[j][q][n][lane], x);
                if (S.shaped) shape<true>(a, S, x, r, at, h);   // (the sums are fp32 whatever the queries)
                if (!r0.there || !r1.there || !B.whole(s.pre, at, 32)) mask(x, seen(a, s, r, at, h, r0.there, r1.there));
                const float l = M.lse[j][lane];
                // (past the last row the columns repeat it: they count for nothing)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], S.c, -l));
                    sum[i] += r.valid ? w : 0.0f;
                }
            }
        }
    }
    // over the 32 columns
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const float v = row16_sum(sum[i]);
        sum[i] = v + swap16_other(v);
    }
    if ((lane & 31) != 0) return;
    const int64_t row = (int64_t)pair * a.max_len;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int p = at + pos32(i, h);
        if (p >= a.max_len) continue;
        if (a.mass_parts > 1) {
            a.mass_part[((int64_t)part * pairs) * a.max_len + row + p] = sum[i];
            continue;
        }
        const float was = a.mass && p < a.mass_width ? a.mass[pair * a.mass_stride + p] : 0.0f;
        a.mass_out[row + p] = p < s.len ? was + sum[i] : 0.0f;
    }
}

}  // namespace

#define SMX_PG_NAME_(f, w, b) f##_w##w##_b##b
#define SMX_PG_NAME(f, w, b) SMX_PG_NAME_(f, w, b)
hipError_t SMX_PG_NAME(launch_attn_mass, SMX_PG_W, SMX_PG_BF16)(const AttnPgArgs &a, const MassPgPlan &p, hipStream_t s)
{
    const unsigned n = (unsigned)p.blocks;
    if (a.io == PG_F32) k_attn_mass<true><<<n, kWaves * 64, 0, s>>>(a);
    else k_attn_mass<false><<<n, kWaves * 64, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
