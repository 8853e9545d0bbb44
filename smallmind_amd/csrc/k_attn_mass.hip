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
//
// What bounds it.  Few rows: memory, after the chain from page table to rows (16 sequences of up to 1024 positions, 32 heads of 64:
// 13 us, of which 46 MB take 7).  Many rows (4095 tokens, 32 heads over 8 of 128: 115 us with the join's 7; the products alone would
// take 56): some 8600 clocks of a SIMD for 128 rows and a wave's 64 positions, the vector unit busy for 36 of 100 and the matrix cores
// for 24.  Of 2048 workgroups 1088 lie on the visible side, 2.1 times what the chip holds; what else is waited for was not measured.  fp32
// queries, two or three parts, leave one wave on a SIMD there: 309 us over an F16 cache, 439 over a BF16 one.
#include "smx_attn_paged_dev.h"

namespace smx {

namespace {

constexpr int kWaves = 4;
constexpr int KT = W <= 128 ? 2 : 1;      // 32-position groups of a wave (many rows)
constexpr int kKeys = 32 * KT * kWaves;   // positions of a workgroup

// The sums over a wave's 32 columns, element i's in lanes 32 h + i and 32 h + 16 + i: every exchange halves the elements that a lane
// still adds up, keeping those whose number has the lane's bit (48 instructions; sixteen sums one by one, 112).
__device__ __forceinline__ float pick(uint32_t m, float a, float b)   // m all ones: a, 0: b
{
    return __uint_as_float((__float_as_uint(a) & m) | (__float_as_uint(b) & ~m));
}
__device__ __forceinline__ float sum_columns(const float16v &x, int lane)
{
    const uint32_t m8 = -(uint32_t)(lane >> 3 & 1), m4 = -(uint32_t)(lane >> 2 & 1), m2 = -(uint32_t)(lane >> 1 & 1), m1 = -(uint32_t)(lane & 1);
    float v[8], w[4], z[2];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = pick(m8, x[i + 8], x[i]) + dpp_mov<0x128>(pick(m8, x[i], x[i + 8]));   // from lane ^ 8
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int lo = i + (i & 2);   // 0 1 4 5
        w[i] = pick(m2, v[lo + 2], v[lo]) + dpp_mov<0x4E>(pick(m2, v[lo], v[lo + 2]));                        // lane ^ 2
    }
#pragma unroll
    for (int i = 0; i < 2; i++) z[i] = pick(m1, w[2 * i + 1], w[2 * i]) + dpp_mov<0xB1>(pick(m1, w[2 * i], w[2 * i + 1]));   // lane ^ 1
    const float r = pick(m4, z[1], z[0]) + __shfl_xor(pick(m4, z[0], z[1]), 4, 64);
    return r + swap16_other(r);
}

// What the positions of 32 from `at` on have received, as sum_columns leaves it.
struct Giving {
    int p;
    float was;
    __device__ __forceinline__ Giving(const AttnPgArgs &a, int pair, int at, int lane)   // (asked early: what there was is on its way)
    {
        p = lane & 16 ? a.max_len : at + pos32(lane & 15, lane >> 5);
        was = a.mass_parts == 1 && a.mass && p < a.mass_width && p < a.max_len ? a.mass[pair * a.mass_stride + p] : 0.0f;
    }
    __device__ __forceinline__ void give(const AttnPgArgs &a, const Seq &s, int pair, int part, float v) const
    {
        if (p >= a.max_len) return;
        const int64_t at = (int64_t)pair * a.max_len + p;
        if (a.mass_parts > 1) a.mass_part[(int64_t)part * a.n_seq * a.c.n_kv * a.max_len + at] = v;
        else a.mass_out[at] = p < s.len ? was + v : 0.0f;
    }
};

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

// lse of a row as an exponent of 2: l is what the table has.
__device__ __forceinline__ float lse_of(const Row &r, float l)
{
    // (a row that sees nothing has -inf; one past the last repeats that one and counts for nothing)
    return !r.valid ? __builtin_huge_valf() : l == -__builtin_huge_valf() ? 0.0f : l * 1.4426950408889634f;
}

// A row whose lse is NaN (its query, or a position that it sees, is not finite) gives NaN to what it sees and nothing to the rest:
// its products are NaN, and masked before lse is taken off.
template <bool F32>
__device__ __forceinline__ void settle(Query<F32> &Q, float &lse)
{
    const bool bad = lse != lse;
    spoil(Q, bad);
    if (bad) lse = 0.0f;
}

// ---- few rows ----------------------------------------------------------------------------------------
// A workgroup takes a share of a sequence's positions, 32 at a time in turn with its other waves.
template <bool F32>
__global__ __launch_bounds__(kWaves * 64) void k_attn_mass_few(const AttnPgArgs a)
{
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const int pairs = a.n_seq * a.c.n_kv, shares = gridDim.x / pairs, head = blockIdx.x % a.c.n_kv, rest = blockIdx.x / a.c.n_kv;
    const int b = a.ranked ? nth_longest(a, rest / shares) : rest % a.n_seq, share = a.ranked ? rest % shares : rest / a.n_seq;
    const int pair = b * a.c.n_kv + head;
    const Seq s = seq_of(a, b);
    const int step = 32 * kWaves * shares;
    int at = 32 * (kWaves * share + wave);
    elem8 k[2][NK];
    bool there[2][2];
    const bool any_rows = s.rows > 0;
    if (any_rows && at < s.len) {
        Pages P(a, s, head, at / kPgGroup);
        load_k(a, s, P, at, lane, k[0], there[0][0], there[0][1]);
        const Row r = row_of(a, s, head, lane & 31);
        float lse = a.lse_in[(int64_t)r.token * a.n_head + r.head];
        Query<F32> Q;
        load_q<F32, false>(a, r, h, Q);   // (a row that is not finite has an lse of NaN)
        settle(Q, lse);
        lse = lse_of(r, lse);
        const Shape S(a, a.slopes ? a.slopes[r.head] : 0.0f, Q.unit);
        const Bounds B = bounds_of(a, s, s.first, row_of(a, s, head, s.rows - 1).t);
        const auto go = [&](const elem8 (&kk)[NK], bool th0, bool th1, elem8 (&next)[NK], bool (&th)[2]) {
            const Giving G(a, pair, at, lane);
            if (at + step < s.len) load_k(a, s, P, at + step, lane, next, th[0], th[1]);
            float sum;
            if (B.none(s.pre, at, 32)) {
                sum = 0.0f;
            } else {
                float16v x;
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int q = 0; q < kParts<F32>; q++) x = mfma(kk[n], Q.q[q][n], n || q ? x : float16v(0.0f));
                if (S.shaped) shape<false>(a, S, x, r.t, at, h);   // (the sums are fp32 whatever the queries)
                if (!th0 || !th1 || !B.whole(s.pre, at, 32)) mask(x, seen(a, s, r.t, at, h, th0, th1));
#pragma unroll
                for (int i = 0; i < 16; i++) x[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], S.c, -lse));
                sum = sum_columns(x, lane);
            }
            G.give(a, s, pair, 0, sum);
            at += step;
        };
        while (at < s.len) {
            go(k[0], there[0][0], there[0][1], k[1], there[1]);
            if (at < s.len) go(k[1], there[1][0], there[1][1], k[0], there[0]);
        }
    }
    // positions that nobody is there to see: what they had; 0 beyond the sequence
    for (int p = (any_rows ? (s.len + 31) / 32 * 32 : 0) + share * kWaves * 64 + (int)threadIdx.x; p < a.max_len; p += shares * kWaves * 64)
        a.mass_out[(int64_t)pair * a.max_len + p] = p < s.len && a.mass && p < a.mass_width ? a.mass[pair * a.mass_stride + p] : 0.0f;
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
    constexpr bool FAST = NB == 4;   // (with fewer, registers are short)
    const bool shaped = a.cap_in != 0.0f || a.slopes;
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
    const int first = t_lo * a.group, blocks = k0 < s.len ? max(0, (t_hi * a.group - first + 32 * NB - 1) / (32 * NB)) : 0;   // of NB * 32 rows
    const int s0 = part * a.mass_per, s1 = min(blocks, s0 + a.mass_per);
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
        float lse = 0.0f, slope = 0.0f;   // as loaded: nothing here is to wait for what has just been asked for
        Row r{};
        const auto fetch = [&](int st) {
            r = row_of(a, s, head, first + (st * NB + wave) * 32 + (lane & 31));
            load_q<F32, false>(a, r, h, Q);   // (a row that is not finite has an lse of NaN)
            lse = a.lse_in[(int64_t)r.token * a.n_head + r.head];
            if (a.slopes) slope = a.slopes[r.head];
        };
        if (wave < NB) fetch(s0);
        // K has landed: otherwise the compiler, which does not know, has every turn wait for the rows just asked for
        wait_loads<0>();
        for (int st = s0; st < s1; st++) {
            __syncthreads();   // the rows before have been read
            if (wave < NB) {
                settle(Q, lse);
#pragma unroll
                for (int q = 0; q < NP; q++)
#pragma unroll
                    for (int n = 0; n < NK; n++) M.q[wave][q][n][lane] = Q.q[q][n];
                if (h == 0) {
                    const Shape S(a, slope, Q.unit);
                    M.in[wave][lane] = S.in, M.slope[wave][lane] = S.slope, M.lse[wave][lane] = lse_of(r, lse), M.t[wave][lane] = r.t;
                }
            }
            __syncthreads();
            if (wave < NB && st + 1 < s1) fetch(st + 1);
            const int row0 = first + st * 32 * NB, c = lane & 31;
            if (at >= s.len) continue;
            const auto scores = [&](float16v (&x)[KT], int j) {
#pragma unroll
                for (int n = 0; n < NK; n++)
#pragma unroll
                    for (int q = 0; q < NP; q++) {
                        const elem8 qq = M.q[j][q][n][lane];
#pragma unroll
                        for (int u = 0; u < KT; u++) x[u] = mfma(k[u][n], qq, n || q ? x[u] : float16v(0.0f));
                    }
            };
            const auto add = [&](const float16v (&x)[KT], float by, float l) {
#pragma unroll
                for (int u = 0; u < KT; u++)
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[u][i] += __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][i], by, -l));
            };
            if constexpr (FAST) {
                // every row sees all of the wave's positions: no bounds to look at, and the next rows' scores beside these ones' weights
                const Bounds B = bounds_of(a, s, M.t[0][0], M.t[NB - 1][31]);
                if (!shaped && all && row0 + 32 * NB <= s.rows && B.whole(s.pre, at, 32 * KT)) {
                    float16v x[2][KT];
                    scores(x[0], 0);
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        __builtin_amdgcn_sched_barrier(0);
                        if (j + 1 < NB) scores(x[(j + 1) & 1], j + 1);
                        add(x[j & 1], M.in[j][c], M.lse[j][c]);
                        constexpr int MK = NK * NP * KT, E = 16 * KT;   // matrix instructions, elements
                        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                        for (int i = 0; i < MK; i++) {
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            if (i % KT == 0) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x002, (2 * E + MK - 1) / MK, 0);
                            __builtin_amdgcn_sched_group_barrier(0x400, (E + MK - 1) / MK, 0);
                        }
                    }
                    continue;
                }
            }
            for (int j = 0; j < NB; j++) {
                if (row0 + 32 * j >= s.rows) break;
                const int t = M.t[j][c];
                const Bounds B = bounds_of(a, s, t, __builtin_amdgcn_readlane(t, 31));
                if (B.none(s.pre, at, 32 * KT)) continue;
                Shape S;
                S.shaped = shaped;
                S.in = M.in[j][c], S.slope = M.slope[j][c], S.c = shaped ? 1.0f : S.in;
                float16v x[KT];
                scores(x, j);
                if (shaped) {
#pragma unroll
                    for (int u = 0; u < KT; u++) shape<false>(a, S, x[u], t, at + 32 * u, h);   // (the sums are fp32 whatever the queries)
                }
                if (!all || !B.whole(s.pre, at, 32 * KT)) {
#pragma unroll
                    for (int u = 0; u < KT; u++) mask(x[u], seen(a, s, t, at + 32 * u, h, there[u][0], there[u][1]));
                }
                add(x, S.c, M.lse[j][c]);
            }
        }
    }
#pragma unroll
    for (int u = 0; u < KT; u++) Giving(a, pair, at + 32 * u, lane).give(a, s, pair, part, sum_columns(sum[u], lane));
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
