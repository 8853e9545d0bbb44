// k_attn_paged.hip -- attention of a ragged batch of new tokens over the paged KV cache (smx_paged.h): chunks of prompts
// and single tokens in one call.  Built once per row width and element type.
//
// Mathematics.  A row is one query head of one token.  With s = scale q . k (or cap tanh(s / cap)), less slope |t - p|, as an
// exponent of 2, and the running maximum m of s over the positions p that the row sees,
//     out = sum_p 2^(s_p - m) v_p / sum_p 2^(s_p - m),
// one pass over the positions.  m moves only where a maximum has grown by more than 2^8, so that the sums are seldom rescaled.
// Sums are fp32.  16-bit queries and weights are the matrix instructions' own operands (a weight rounded to the type of the
// output it ends in); fp32 queries and weights go in as parts: two of fp16, 22 bits, after a power of two has brought a
// row's largest to the range of fp16, three of bf16, 24 bits.
//
// Layout.  A wave computes S^T = K q^T on 32x32x16 matrix instructions: lane 32 h + c gets row c's scores of the positions
// 8 (i / 4) + 4 h + i % 4 of 32, and these are the positions that it brings to the second product out^T = V^T w^T, whose V operand is
// read out of LDS transposed, in that order: weights do not move between lanes, a row's maximum and sum take one exchange.
//
// Two ways through the positions, in chunks of one workgroup each; k_attn_paged_join adds up what the chunks found.
//   many rows: a block of 128 or 256 rows of one sequence and KV head (the group's heads of a token are neighbouring rows), 32 per
//     wave; all walk the same tiles of 64 positions, which go from memory to LDS one tile ahead.
//   few rows (up to 32 per KV head): every wave holds all of them and takes tiles of 32 positions in turn, K from memory to
//     registers, V to LDS of its own; the waves join their sums at the end.
#include "smx_attn_paged_dev.h"

namespace smx {

namespace {

// A weight is 2^(s - m + kOff): fp16 then holds weights down to 2^-30 of the largest, and up to 2^8 above it (kLazy), to
// full precision; bf16 has the range of fp32.
constexpr float kOff = BF16 ? 0.0f : 6.0f;
constexpr float kLazy = 8.0f;

// ---- the running softmax of 32 rows, a row per column of two lanes ---------------------------------
struct Running {
    // weights so far are 2^(x c + b); m: the x that b was taken from (-inf: nothing seen), l: this lane's share of their sum
    float m = kNegInf, b = 0.0f, l = 0.0f;
    float16v acc[ND];

    __device__ __forceinline__ Running()
    {
#pragma unroll
        for (int n = 0; n < ND; n++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[n][i] = 0.0f;
    }

    // x of KT * 32 positions become weights' parts: w[part][16 positions].
    template <int KT, int NP>
    __device__ __forceinline__ void step(float16v (&x)[KT], float c, elem8 (&w)[NP][2 * KT])
    {
        float top = x[0][0];
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int i = 0; i < 16; i++) top = fmaxf(top, x[t][i]);
        top = max_halves(top);
        // (nothing seen yet: m = -inf, and the difference NaN or inf)
        const bool grown = top > kNegInf && !((top - m) * c <= kLazy);
        if (__any(grown)) {
            const float was = b;
            if (grown) {
                const bool none = m == kNegInf;
                m = top;
                b = kOff - m * c;
                const float f = none ? 0.0f : __builtin_amdgcn_exp2f(b - was);
                l *= f;
#pragma unroll
                for (int n = 0; n < ND; n++) acc[n] *= f;
            }
        }
        // x c + b in one rounding: b's own is the same for all of a row's weights.  It passes 1 where scores pass 2^24, whose
        // products are not known better than that either, but there a weight could overflow.
        float e = b;
        if (__any(fabsf(b) > 16777216.0f)) {
            if (fabsf(b) > 16777216.0f) {
#pragma unroll
                for (int t = 0; t < KT; t++)
#pragma unroll
                    for (int i = 0; i < 16; i++) x[t][i] -= m;
                e = kOff;
            }
        }
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[t][i], c, e));
                sum += p;
                elem s[NP];
                split(p, s);
#pragma unroll
                for (int k = 0; k < NP; k++) w[k][2 * t + (i >> 3)][i & 7] = s[k];
            }
        }
        l += sum;
    }
};

// Outputs of a wave's 32 rows, or their part of them.
template <bool F32>
__device__ __forceinline__ void finish(const AttnPgArgs &a, const Running &R, const Row &r, int h, int part)
{
    const float sum = sum_halves(R.l);
    if (!r.valid) return;
    const int64_t id = (int64_t)r.token * a.n_head + r.head;
    const bool none = R.m == kNegInf && sum == 0.0f;   // (a sum of NaN: NaN was seen)
    if (a.parts > 1) {
        const int64_t at = (int64_t)part * a.n_tok * a.n_head + id;
        if (h == 0) a.part_ml[2 * at] = none ? kNegInf : -R.b, a.part_ml[2 * at + 1] = sum;
        float *dst = a.part_acc + at * a.c.hd + 4 * h;
#pragma unroll
        for (int n = 0; n < ND; n++)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                if (32 * n + 2 * i + 4 * h < a.c.hd)
                    *(float4 *)(dst + 32 * n + 2 * i) = make_float4(R.acc[n][i], R.acc[n][i + 1], R.acc[n][i + 2], R.acc[n][i + 3]);
        return;
    }
    if (a.lse && h == 0) a.lse[id] = none ? kNegInf : (__builtin_amdgcn_logf(sum) - R.b) * 0.69314718055994531f;
    const float inv = none ? 0.0f : 1.0f / sum;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = 32 * n + 2 * i + 4 * h;
            if (d >= a.c.hd) continue;
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = none ? 0.0f : R.acc[n][i + e] * inv;
            if constexpr (F32) {
                float *dst = (float *)a.out + id * a.c.hd + d;
                if (a.out_vec) {
                    *(float4 *)dst = make_float4(o[0], o[1], o[2], o[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) dst[e] = o[e];
                }
            } else {
                elem *dst = (elem *)a.out + id * a.c.hd + d;
                const elem4 v = {(elem)o[0], (elem)o[1], (elem)o[2], (elem)o[3]};
                if (a.out_vec) {
                    *(elem4 *)dst = v;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) dst[e] = v[e];
                }
            }
        }
}

// Rows without a part here: no weight.
__device__ __forceinline__ void finish_empty(const AttnPgArgs &a, const Row &r, int h, int part)
{
    if (!r.valid || h) return;
    const int64_t at = (int64_t)part * a.n_tok * a.n_head + (int64_t)r.token * a.n_head + r.head;
    a.part_ml[2 * at] = kNegInf, a.part_ml[2 * at + 1] = 0.0f;
}

// ---- many rows -------------------------------------------------------------------------------------
struct Tile {
    uint8_t k[kPgTile * ROW], v[kPgTile * ROW];
};

// A tile of positions on its way to LDS: each of NW waves brings a share of its kilobytes.
template <int NW>
__device__ __forceinline__ void bring(const AttnPgArgs &a, const Seq &s, int head, int tile, Tile &T, int wave, int lane)
{
    constexpr int PER = W / 32;   // kilobytes of 16 rows
#pragma unroll
    for (int i0 = 0; i0 < 4 * PER; i0 += NW) {
        const int i = i0 + wave;
        if (4 * PER % NW != 0 && i >= 4 * PER) break;
        const int b = i / PER, off = b * 16 * ROW + (i - b * PER) * 1024;
        const uint8_t *src = rows16(a, s, head, 4 * tile + b).p + (i - b * PER) * 1024 + lane * 16;
        to_lds(src, T.k + off);
        to_lds(src + a.c.v_off(), T.v + off);
    }
}

template <bool F32, int NW>
__device__ __forceinline__ void many(const AttnPgArgs &a, Tile (&T)[2], const Seq &s, int head, int row0, int part)
{
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const int mine = row0 + wave * kPgRows;
    const int t0 = row_of(a, s, head, row0).t, t1 = row_of(a, s, head, row0 + NW * kPgRows - 1).t;
    const Range rg = range_of(a, s, __builtin_amdgcn_readfirstlane(t0), __builtin_amdgcn_readfirstlane(t1));
    const int i0 = part * a.chunk, i1 = a.parts > 1 ? min(rg.count, i0 + a.chunk) : rg.count;
    const Row r = row_of(a, s, head, mine + (lane & 31));
    const bool busy = mine < s.rows;   // (a wave without rows brings its share of the tiles)
    if (i0 >= i1) {
        if (a.parts > 1) { if (busy) finish_empty(a, r, h, part); return; }
        Running R;
        if (busy) finish<F32>(a, R, r, h, part);
        return;
    }
    bring<NW>(a, s, head, rg.tile(i0), T[0], wave, lane);
    Query<F32> Q;
    load_q<F32>(a, r, h, Q);
    const Shape S(a, r, Q.unit);
    const Bounds B = bounds_of(a, s, mine, kPgRows);
    const LaneAt L(lane);
    constexpr int KT = W * kParts<F32> > 512 ? 1 : 2;   // 32-position halves of a tile at once: two where registers suffice
    Running R;
    for (int i = i0; i < i1; i++) {
        const int tile = rg.tile(i), at = tile * kPgTile;
        wait_all();
        __syncthreads();   // this tile is there, the one before has been read
        if (i + 1 < i1) bring<NW>(a, s, head, rg.tile(i + 1), T[(i + 1 - i0) & 1], wave, lane);
        if (!busy || B.none(s.pre, at, kPgTile)) continue;
        const Tile &C = T[(i - i0) & 1];
        bool there[4], all = true;
#pragma unroll
        for (int b = 0; b < 4; b++) there[b] = rows16(a, s, head, 4 * tile + b).there, all = all && there[b];
        const bool cut = !all || !B.whole(s.pre, at, kPgTile);
#pragma unroll
        for (int t0 = 0; t0 < 2; t0 += KT) {
            float16v x[KT];
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int e = 0; e < 16; e++) x[t][e] = 0.0f;
#pragma unroll
            for (int n = 0; n < NK; n++)
#pragma unroll
                for (int t = 0; t < KT; t++) {
                    const elem8 k = L.key(C.k + (t0 + t) * 32 * ROW, n);
#pragma unroll
                    for (int p = 0; p < kParts<F32>; p++) x[t] = mfma(k, Q.q[p][n], x[t]);
                }
            if (S.shaped) {
#pragma unroll
                for (int t = 0; t < KT; t++) shape(a, S, x[t], r, at + 32 * (t0 + t), h);
            }
            if (cut) {
#pragma unroll
                for (int t = 0; t < KT; t++) mask(x[t], r, s.pre, at + 32 * (t0 + t), h, there[2 * (t0 + t)], there[2 * (t0 + t) + 1]);
            }
            elem8 w[kParts<F32>][2 * KT];
            R.step<KT, kParts<F32>>(x, S.c, w);
#pragma unroll
            for (int b = 0; b < 2 * KT; b++)
#pragma unroll
                for (int d = 0; d < ND; d++) {
                    const elem8 v = L.val(C.v + (2 * t0 + b) * 16 * ROW, d);
#pragma unroll
                    for (int p = 0; p < kParts<F32>; p++) R.acc[d] = mfma(v, w[p][b], R.acc[d]);
                }
        }
    }
    if (busy) finish<F32>(a, R, r, h, part);
}

// ---- few rows --------------------------------------------------------------------------------------
// Memory of NW waves: V of 32 positions twice for each, then the joining of their sums.
template <int NW> union Few {
    uint8_t v[NW][2][32 * ROW];
    struct {
        float m[NW / 2][64], b[NW / 2][64], l[NW / 2][64];
        float acc[NW / 2][ND * 16][64];
    } j;
};

// `of` added to R.
__device__ __forceinline__ void join(Running &R, float m, float b, float l, const float (*acc)[64], int lane)
{
    // the higher of the two references; one without weight brings nothing
    const bool none = m == kNegInf && l == 0.0f;
    const bool up = !none && (R.m == kNegInf || b < R.b);
    const float nb = up ? b : R.b;
    const float f = R.m == kNegInf && R.l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(nb - R.b), g = none ? 0.0f : __builtin_amdgcn_exp2f(nb - b);
    R.l = R.l * f + l * g;
#pragma unroll
    for (int n = 0; n < ND; n++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float o = acc[n * 16 + i][lane];
            R.acc[n][i] = R.acc[n][i] * f + (none ? 0.0f : o * g);
        }
    if (up) R.m = m;
    R.b = nb;
}

template <bool F32, int NW>
__device__ __forceinline__ void few(const AttnPgArgs &a, Few<NW> &F, const Seq &s, int head, int part)
{
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const Row r = row_of(a, s, head, lane & 31);
    const Row last = row_of(a, s, head, s.rows - 1);
    const Range rg = range_of(a, s, s.first, __builtin_amdgcn_readfirstlane(last.t));
    // halves of tiles
    const int i0 = 2 * part * a.chunk, i1 = a.parts > 1 ? min(2 * rg.count, i0 + 2 * a.chunk) : 2 * rg.count;
    if (i0 >= i1) {
        if (wave) return;
        if (a.parts > 1) { finish_empty(a, r, h, part); return; }
        Running R;
        finish<F32>(a, R, r, h, part);
        return;
    }
    const auto pos_of = [&](int i) { return rg.tile(i >> 1) * kPgTile + 32 * (i & 1); };
    const uint32_t row_at = (lane & 15) * ROW;
    elem8 k[NK];
    Rows16 r0{}, r1{};
    const auto find = [&](int i) {
        const int blk = pos_of(i) / kPgGroup;
        r0 = rows16(a, s, head, blk), r1 = rows16(a, s, head, blk + 1);
    };
    const auto fetch_k = [&]() {
        const uint8_t *p = (lane & 16 ? r1.p : r0.p) + row_at;
#pragma unroll
        for (int n = 0; n < NK; n++) k[n] = *(const elem8 *)(p + 16 * pg_unit(W, 2 * n + h, lane & 15));
    };
    const auto fetch_v = [&](uint8_t *v) {
#pragma unroll
        for (int j = 0; j < W / 32; j++) {
            to_lds(r0.p + a.c.v_off() + 1024 * j + lane * 16, v + 1024 * j);
            to_lds(r1.p + a.c.v_off() + 1024 * j + lane * 16, v + 16 * ROW + 1024 * j);
        }
    };
    if (i0 + wave < i1) {
        find(i0 + wave);
        fetch_k();
        fetch_v(F.v[wave][0]);
    }
    Query<F32> Q;
    load_q<F32>(a, r, h, Q);
    const Shape S(a, r, Q.unit);
    const Bounds B = bounds_of(a, s, 0, kPgRows);
    const LaneAt L(lane);
    Running R;
    int buf = 0;
    for (int i = i0 + wave; i < i1; i += NW, buf ^= 1) {
        const uint8_t *v = F.v[wave][buf];
        const int at = pos_of(i);
        const bool th0 = r0.there, th1 = r1.there, cut = !th0 || !th1 || !B.whole(s.pre, at, 32), more = i + NW < i1;
        wait_all();
        if (more) {
            find(i + NW);
            fetch_v(F.v[wave][buf ^ 1]);
        }
        float16v x[1];
#pragma unroll
        for (int e = 0; e < 16; e++) x[0][e] = 0.0f;
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int p = 0; p < kParts<F32>; p++) x[0] = mfma(k[n], Q.q[p][n], x[0]);
        if (more) fetch_k();
        if (B.none(s.pre, at, 32)) continue;
        if (S.shaped) shape(a, S, x[0], r, at, h);
        if (cut) mask(x[0], r, s.pre, at, h, th0, th1);
        elem8 w[kParts<F32>][2];
        R.step<1, kParts<F32>>(x, S.c, w);
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const elem8 vv = L.val(v + b * 16 * ROW, d);
#pragma unroll
                for (int p = 0; p < kParts<F32>; p++) R.acc[d] = mfma(vv, w[p][b], R.acc[d]);
            }
    }
    // the waves' sums, half of them handing theirs to the other half
#pragma unroll
    for (int n = NW / 2; n >= 1; n /= 2) {
        __syncthreads();
        if (wave >= n && wave < 2 * n) {
            F.j.m[wave - n][lane] = R.m, F.j.b[wave - n][lane] = R.b, F.j.l[wave - n][lane] = R.l;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) F.j.acc[wave - n][d * 16 + i][lane] = R.acc[d][i];
        }
        __syncthreads();
        if (wave < n) join(R, F.j.m[wave][lane], F.j.b[wave][lane], F.j.l[wave][lane], F.j.acc[wave], lane);
    }
    if (wave == 0) finish<F32>(a, R, r, h, part);
}

// Finds the block's sequence.  Block x belongs to the last sequence whose first block floor(start * group / rows) + b is
// not above x: no sequence has more blocks than lie between its own first and the next one's.
template <bool F32, int NW>
__device__ __forceinline__ void many_rows(const AttnPgArgs &a, Tile (&T)[2])
{
    const int pairs = a.c.n_kv * a.parts;
    const int block = a.tile_blocks - 1 - (int)blockIdx.x / pairs, pair = (int)blockIdx.x % pairs;
    const int lane = threadIdx.x & 63;
    int b = -1;
    for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
        const int i = min(b0 + lane, a.n_seq - 1);
        const int64_t first = (int64_t)min(max(a.starts[i], 0), a.n_tok) * a.group / (NW * kPgRows) + i;
        const int n = __popcll(__ballot(b0 + lane < a.n_seq && first <= block));
        b += n;
        if (n < 64) break;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b < 0) return;
    const Seq s = seq_of(a, b);
    const int64_t first = (int64_t)s.start * a.group / (NW * kPgRows) + b;
    const int64_t row0 = (block - first) * (NW * kPgRows);
    if (row0 >= s.rows || s.rows <= a.short_rows) return;
    many<F32, NW>(a, T, s, pair % a.c.n_kv, (int)row0, pair / a.c.n_kv);
}

// Workgroups [0, tile_wgs): blocks of NW * 32 rows (KV head and part fastest, the last blocks, which see most, first); the others: a
// short sequence each.  MANY: there are any of the former.
template <bool F32, bool MANY, int NW>
__global__ __launch_bounds__(NW * 64, !MANY && W <= 128 && W * kParts<F32> <= 256 ? 2 : 1) void k_attn_paged(const AttnPgArgs a)
{
    union Mem {
        Tile tiles[MANY ? 2 : 1];
        Few<NW> few;
    };
    __shared__ __align__(1024) char mem[MANY ? sizeof(Mem) : sizeof(Few<NW>)];
    Mem &M = *(Mem *)mem;
    if constexpr (MANY) {
        if ((int)blockIdx.x < a.tile_wgs) {
            many_rows<F32, NW>(a, M.tiles);
            return;
        }
    }
    const int i = blockIdx.x - a.tile_wgs, units = a.n_seq * a.c.n_kv, unit = i % units;
    const Seq s = seq_of(a, unit / a.c.n_kv);
    if (s.rows <= 0 || s.rows > kPgRows) return;
    few<F32, NW>(a, M.few, s, unit % a.c.n_kv, i / units);
}

// Waves of the blocks of many rows: eight where their registers suffice (256 a lane), else four (512).
template <bool F32> constexpr int kManyWaves = W * (1 + kParts<F32>) <= 256 ? 8 : 4;

template <bool F32>
hipError_t launch(const AttnPgArgs &a, const AttnPgPlan &p, hipStream_t s)
{
    const unsigned n = (unsigned)p.blocks;
    if (p.kind == 0) k_attn_paged<F32, false, 4><<<n, 256, 0, s>>>(a);
    else if (p.kind == 1) k_attn_paged<F32, true, 4><<<n, 256, 0, s>>>(a);
    else if constexpr (kManyWaves<F32> == 8) k_attn_paged<F32, true, 8><<<n, 512, 0, s>>>(a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

#define SMX_PG_NAME_(f, w, b) f##_w##w##_b##b
#define SMX_PG_NAME(f, w, b) SMX_PG_NAME_(f, w, b)
hipError_t SMX_PG_NAME(launch_attn_paged, SMX_PG_W, SMX_PG_BF16)(const AttnPgArgs &a, const AttnPgPlan &p, hipStream_t s)
{
    return a.io == PG_F32 ? launch<true>(a, p, s) : launch<false>(a, p, s);
}
int SMX_PG_NAME(attn_paged_waves, SMX_PG_W, SMX_PG_BF16)(int io) { return io == PG_F32 ? kManyWaves<true> : kManyWaves<false>; }

}  // namespace smx
