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
//   many rows: a block of 128 rows of one sequence and KV head (the group's heads of a token are neighbouring rows), 32 per
//     wave; all walk the same tiles of 64 positions, which go from memory to LDS one tile ahead (PgMode).
//   few rows (up to 32 per KV head): every wave holds all of them and takes tiles of 32 positions in turn, K from memory to
//     registers, V to LDS of its own; the waves join their sums at the end.
//
// What bounds it.  Many rows of 128 dims: the matrix cores, at the clock that the card's power leaves them (2048 tokens over
// 32768 positions, 32 heads over 8, bf16: 970 to 1090 us, 980 to 1100 TFLOP/s, where the library's product of 8192^3 reaches
// 1160 to 1225).  64 dims: the vector unit's 32 exponentials and some 110 other instructions of a wave's tile beside 16 matrix
// instructions (4096 over 16384, 32 heads over 8: 585 to 620 us, 780 to 820 TFLOP/s); a cap adds 5 instructions, two of them transcendental,
// to each of 32 scores, slopes 3.  Short prompts: the way in and out of a block and the tiles that the diagonal cuts (4 of
// 1023, 12 heads of 64: 23 us).  fp32 queries over an F16 cache: twice the matrix instructions and the splitting of weights
// (512 over 4096, 32 heads over 4 of 64: 49 us with the join's 6; over a BF16 cache, three times, 71).  Few rows: memory (64 sequences of up to 8192 positions, 8
// heads of 128: 242 us, 5.6 TB/s), in short contexts the chain from page table to rows to the waves' joining (700 positions:
// 10.6 us).
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

    // Moves the reference to what x of KT * 32 positions holds, where that calls for it; returns e: their weights are 2^(x c + e).
    template <int KT>
    __device__ __forceinline__ float refer(float16v (&x)[KT], float c)
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
        return e;
    }

    // x of 32 positions becomes weights' parts: w[part][16 positions].
    template <int NP>
    __device__ __forceinline__ void weigh(const float16v &x, float c, float e, elem8 (&w)[NP][2])
    {
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], c, e)), q = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i + 1], c, e));
            l += p;
            l += q;
            elem2 s[NP];
            split(p, q, s);
#pragma unroll
            for (int k = 0; k < NP; k++) w[k][i >> 3][i & 7] = s[k][0], w[k][i >> 3][(i & 7) + 1] = s[k][1];
        }
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

// What N waves hand to as many others, a value per lane.
template <int N> struct Handed {
    float m[N][64], b[N][64], l[N][64];
    float acc[N][ND * 16][64];

    __device__ __forceinline__ void put(int i, int lane, const Running &R)
    {
        m[i][lane] = R.m, b[i][lane] = R.b, l[i][lane] = R.l;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][d * 16 + e][lane] = R.acc[d][e];
    }
    // added to R
    __device__ __forceinline__ void join(int i, int lane, Running &R) const
    {
        // the higher of the two references; one without weight brings nothing
        const float om = m[i][lane], ob = b[i][lane], ol = l[i][lane];
        const bool none = om == kNegInf && ol == 0.0f, up = !none && (R.m == kNegInf || ob < R.b);
        const float nb = up ? ob : R.b;
        const float f = R.m == kNegInf && R.l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(nb - R.b), g = none ? 0.0f : __builtin_amdgcn_exp2f(nb - ob);
        R.l = R.l * f + ol * g;
#pragma unroll
        for (int n = 0; n < ND; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float o = acc[i][n * 16 + e][lane];
                R.acc[n][e] = R.acc[n][e] * f + (none ? 0.0f : o * g);
            }
        if (up) R.m = om;
        R.b = nb;
    }
};

// ---- many rows -------------------------------------------------------------------------------------
// A wave's share (of four) of the kilobytes of a tile's K, and as much of its V: where they are, and the way to LDS.
struct Share {
    static constexpr int PER = W / 32, N = PER;   // kilobytes of 16 rows; of a wave
    const uint8_t *src[N];

    __device__ __forceinline__ void find(const AttnPgArgs &a, const Pages &P, int tile, int wave)
    {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int i = j * 4 + wave, b = i / PER;
            src[j] = P.rows(a, 4 * tile + b).p + (i - b * PER) * 1024;
        }
    }
    __device__ __forceinline__ void bring(uint8_t *to, size_t off, int wave, int lane) const
    {
#pragma unroll
        for (int j = 0; j < N; j++) {
            to_lds(src[j] + off, lane * 16, to + (j * 4 + wave) * 1024);
        }
    }
};

// Two tiles' K and V.
struct Tiles {
    uint8_t k[2][kPgTile * ROW], v[2][kPgTile * ROW];
};
// Those of NG groups of four waves, then what they hand over at the end.
template <int NG> union Many {
    Tiles t[NG];
    Handed<NG == 2 ? 4 : 1> j;
};

// Tells the compiler how to order a block: its N matrix instructions, NP for every READS reads from LDS, with each the ordinary
// and transcendental vector instructions that share the block; two operands are read before them all.
template <int N, int NP, int READS, int VALU, int TRANS>
__device__ __forceinline__ void interleave()
{
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * READS, 0);
#pragma unroll
    for (int i = 0; i < N; i++) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        if (i % NP == 0) __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        if (VALU) __builtin_amdgcn_sched_group_barrier(0x002, VALU, 0);
        if (TRANS) __builtin_amdgcn_sched_group_barrier(0x400, TRANS, 0);
    }
}

// A block of 128 rows, gone through by NG groups of four waves that take tiles in turn.  SPARE: without the registers for
// another tile's scores.
template <bool F32, int NG, bool SPARE, bool QUICK>
__device__ __forceinline__ void many(const AttnPgArgs &a, Many<NG> &M, const Seq &s, int head, int row0, int part)
{
    constexpr int NP = kParts<F32>;
    // 32-position halves of a tile at once: two where registers suffice, and then the next tile's scores while this one's weigh
    constexpr int KT = W * NP > 512 ? 1 : 2;
    constexpr bool AHEAD = KT == 2 && !SPARE;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id() & 3, group = wave_id() >> 2;
    const int mine = row0 + wave * kPgRows;
    Tiles &T = M.t[group];
    const int t0 = row_of(a, s, head, row0).t, t1 = row_of(a, s, head, row0 + 4 * kPgRows - 1).t;
    const Range rg = range_of(a, s, __builtin_amdgcn_readfirstlane(t0), __builtin_amdgcn_readfirstlane(t1));
    // an even share of what there is to go through, but no less than chunk
    const int per = max((rg.count + a.parts - 1) / a.parts, a.chunk), i0 = part * per, i1 = min(rg.count, i0 + per);
    const Row r = row_of(a, s, head, mine + (lane & 31));
    const bool busy = mine < s.rows;   // (a wave without rows brings its share of the tiles)
    if (i0 >= i1) {
        if (!busy || group) return;
        if (a.parts > 1) { finish_empty(a, r, h, part); return; }
        Running R;
        finish<F32>(a, R, r, h, part);
        return;
    }
    const int mine0 = i0 + group;   // this group's first tile
    Pages P(a, s, head, 4 * rg.tile(min(mine0, i1 - 1)));
    Share kv;
    uint32_t there = 0;   // whether the cache has the pages of the tiles on their way, four bits each, the first one's lowest
    const auto bring_k = [&](int i, int to, int bits) {
        const int tile = rg.tile(i);
        P.go(a, s, 4 * tile);
        there |= (uint32_t)(P.ok >> (4 * tile & 63) & 15) << bits;
        kv.find(a, P, tile, wave);
        kv.bring(T.k[to], 0, wave, lane);
    };
    const auto bring_v = [&](int to) { kv.bring(T.v[to], a.c.v_off(), wave, lane); };   // of the K brought last
    if (mine0 < i1) {
        bring_k(mine0, 0, 0);
        bring_v(0);
    }
    if (AHEAD && mine0 + NG < i1) bring_k(mine0 + NG, 1, 4);
    Query<F32> Q;
    load_q<F32>(a, r, h, Q);
    const Shape S(a, a.slopes ? a.slopes[r.head] : 0.0f, Q.unit);
    const Bounds B = bounds_of(a, s, row_of(a, s, 0, mine).t, row_of(a, s, 0, mine + kPgRows - 1).t);
    const LaneAt L(lane);
    Running R;
    const auto scores = [&](float16v (&x)[KT], const uint8_t *k, int t0) {
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int t = 0; t < KT; t++) {
                const elem8 kk = L.key(k + (t0 + t) * 32 * ROW, n);
#pragma unroll
                for (int p = 0; p < NP; p++) x[t] = mfma(kk, Q.q[p][n], n || p ? x[t] : float16v(0.0f));
            }
    };
    const auto sees = [&](int i) { return busy && i < i1 && !B.none(s.pre, rg.tile(i) * kPgTile, kPgTile); };
    const auto add_v = [&](const elem8 (&w)[NP][2], const uint8_t *v) {   // of 32 positions
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const elem8 vv = L.val(v + b * 16 * ROW, d);
#pragma unroll
                for (int p = 0; p < NP; p++) R.acc[d] = mfma(vv, w[p][b], R.acc[d]);
            }
    };
    bool on = sees(mine0);
    // tile i, its scores in x (AHEAD) and its buffers `at`; the next one's scores go to y
    const auto go = [&](int i, float16v (&x)[KT], float16v (&y)[KT], int at) {
        const int pos = rg.tile(i) * kPgTile;   // (past the last tile: not used)
        wait_loads<0>();
        __syncthreads();   // K of the next tile (without AHEAD this one's) and V of this are there, those before have been read
        const uint32_t th = there & 15;
        there >>= 4;
        if (AHEAD) {
            if (i + NG < i1) bring_v(at ^ 1);
            if (i + 2 * NG < i1) bring_k(i + 2 * NG, at, 4);
        } else if (i + NG < i1) {
            bring_k(i + NG, at ^ 1, 0);
            bring_v(at ^ 1);
        }
        const bool cut = th != 15 || !B.whole(s.pre, pos, kPgTile), more = AHEAD && sees(i + NG);
        if (!more) {   // (what y holds is not used: this says so)
#pragma unroll
            for (int t = 0; t < KT; t++) y[t] = float16v(0.0f);
        }
        if (on) {
#pragma unroll
            for (int t0 = 0; t0 < 2; t0 += KT) {
                if (!AHEAD) scores(x, T.k[at], t0);
                if (S.shaped) {
#pragma unroll
                    for (int t = 0; t < KT; t++) shape<QUICK>(a, S, x[t], r.t, pos + 32 * (t0 + t), h);
                }
                if (cut) {
#pragma unroll
                    for (int t = 0; t < KT; t++)
                        mask(x[t], seen(a, s, r.t, pos + 32 * (t0 + t), h, th >> 2 * (t0 + t) & 1, th >> (2 * (t0 + t) + 1) & 1));
                }
                const float e = R.template refer<KT>(x, S.c);
                // vector instructions of the softmax beside the matrix instructions: the first half's beside the next tile's scores,
                // the second half's beside the first half's sums
                constexpr int VALU = 16 * (NP == 1 ? 5 : NP == 2 ? 8 : 16) / 2;   // of 16 elements
                constexpr int MK = 2 * NK * NP, MV = 2 * ND * NP;                   // matrix instructions
                const uint8_t *v = T.v[at] + t0 * 32 * ROW;
                elem8 w[KT][NP][2];
                // (16-bit weights are so few instructions that the whole softmax goes beside the scores: 2048 tokens over 32768
                // positions, 128 dims, 1060 us for 1090)
                constexpr bool BOTH = KT == 2 && NP == 1;
                if (more) {
                    scores(y, T.k[at ^ 1], 0);
                    R.template weigh<NP>(x[0], S.c, e, w[0]);
                    if constexpr (BOTH) R.template weigh<NP>(x[1], S.c, e, w[1]);
                    interleave<MK, NP, 1, ((1 + BOTH) * VALU + MK - 1) / MK, ((1 + BOTH) * 16 + MK - 1) / MK>();
                } else {
                    R.template weigh<NP>(x[0], S.c, e, w[0]);
                    if constexpr (BOTH) R.template weigh<NP>(x[1], S.c, e, w[1]);
                }
                if constexpr (BOTH) {
                    add_v(w[0], v);
                } else if constexpr (KT == 2) {
                    __builtin_amdgcn_sched_barrier(0);
                    add_v(w[0], v);
                    R.template weigh<NP>(x[1], S.c, e, w[1]);
                    interleave<MV, NP, 2, (VALU + MV - 1) / MV, (16 + MV - 1) / MV>();
                    __builtin_amdgcn_sched_barrier(0);
                }
                add_v(w[KT - 1], v + (KT - 1) * 32 * ROW);
                interleave<(1 + BOTH) * MV, NP, 2, 0, 0>();
            }
        } else if (more) {
            scores(y, T.k[at ^ 1], 0);
        }
        on = AHEAD ? more : sees(i + NG);
    };
    float16v x[KT], y[KT];
    if (AHEAD) {
        wait_loads<0>();
        __syncthreads();
        if (on) scores(x, T.k[0], 0);
    }
    for (int i = i0; i < i1; i += 2 * NG) {   // (every wave meets the same barriers)
        go(i + group, x, y, 0);
        if (i + NG < i1) go(i + NG + group, y, x, 1);
    }
    if constexpr (NG == 2) {
        __syncthreads();
        if (group) M.j.put(wave, lane, R);
        __syncthreads();
        if (group) return;
        M.j.join(wave, lane, R);
    }
    // (the row found anew: its numbers need not be kept while the tiles go by)
    if (busy) finish<F32>(a, R, row_of(a, s, head, mine + (opaque_tid() & 31)), opaque_tid() >> 5 & 1, part);
}

// ---- few rows --------------------------------------------------------------------------------------
// Memory of NW waves: V of 32 positions twice for each, then the joining of their sums.
template <int NW> union Few {
    uint8_t v[NW][2][32 * ROW];
    Handed<NW / 2> j;
};

template <bool F32, int NW, bool QUICK>
__device__ __forceinline__ void few(const AttnPgArgs &a, Few<NW> &F, const Seq &s, int head, int part)
{
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = wave_id();
    const Row r = row_of(a, s, head, lane & 31);
    const Row last = row_of(a, s, head, s.rows - 1);
    const Range rg = range_of(a, s, s.first, __builtin_amdgcn_readfirstlane(last.t));
    // halves of tiles
    const int per = 2 * max((rg.count + a.parts - 1) / a.parts, a.chunk), i0 = part * per, i1 = min(2 * rg.count, i0 + per);
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
    Pages P(a, s, head, pos_of(min(i0 + wave, i1 - 1)) / kPgGroup);
    Rows16 r0{}, r1{};
    const auto find = [&](int i) {
        const int blk = pos_of(i) / kPgGroup;
        P.go(a, s, blk);
        r0 = P.rows(a, blk), r1 = P.rows(a, blk + 1);
    };
    const auto fetch_k = [&]() {
        const uint8_t *p = (lane & 16 ? r1.p : r0.p) + row_at;
#pragma unroll
        for (int n = 0; n < NK; n++) k[n] = *(const elem8 *)(p + 16 * pg_unit(W, 2 * n + h, lane & 15));
    };
    const auto fetch_v = [&](uint8_t *v) {
#pragma unroll
        for (int j = 0; j < W / 32; j++) {
            to_lds(r0.p + a.c.v_off() + 1024 * j, lane * 16, v + 1024 * j);
            to_lds(r1.p + a.c.v_off() + 1024 * j, lane * 16, v + 16 * ROW + 1024 * j);
        }
    };
    if (i0 + wave < i1) {
        find(i0 + wave);
        fetch_k();
        fetch_v(F.v[wave][0]);
    }
    Query<F32> Q;
    load_q<F32>(a, r, h, Q);
    const Shape S(a, a.slopes ? a.slopes[r.head] : 0.0f, Q.unit);
    const Bounds B = bounds_of(a, s, s.first, last.t);
    const LaneAt L(lane);
    Running R;
    int buf = 0;
    for (int i = i0 + wave; i < i1; i += NW, buf ^= 1) {
        const uint8_t *v = F.v[wave][buf];
        const int at = pos_of(i);
        const bool th0 = r0.there, th1 = r1.there, cut = !th0 || !th1 || !B.whole(s.pre, at, 32), more = i + NW < i1;
        wait_loads<0>();
        if (more) {
            find(i + NW);
            fetch_v(F.v[wave][buf ^ 1]);
        }
        float16v x[1];
#pragma unroll
        for (int n = 0; n < NK; n++)
#pragma unroll
            for (int p = 0; p < kParts<F32>; p++) x[0] = mfma(k[n], Q.q[p][n], n || p ? x[0] : float16v(0.0f));
        if (more) fetch_k();
        if (B.none(s.pre, at, 32)) continue;
        if (S.shaped) shape<QUICK>(a, S, x[0], r.t, at, h);
        if (cut) mask(x[0], seen(a, s, r.t, at, h, th0, th1));
        elem8 w[kParts<F32>][2];
        const float e = R.refer<1>(x, S.c);
        R.weigh<kParts<F32>>(x[0], S.c, e, w);
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
        if (wave >= n && wave < 2 * n) F.j.put(wave - n, lane, R);
        __syncthreads();
        if (wave < n) F.j.join(wave, lane, R);
    }
    if (wave == 0) finish<F32>(a, R, r, h, part);
}

// Finds the block's sequence.  Block x belongs to the last sequence whose first block floor(start * group / 128) + b is
// not above x: no sequence has more blocks than lie between its own first and the next one's.
template <bool F32, int NG, bool SPARE, bool QUICK>
__device__ __forceinline__ void many_rows(const AttnPgArgs &a, Many<NG> &M)
{
    constexpr int ROWS = 4 * kPgRows;
    // KV head and part fastest; of equal shares of the blocks, one for each sequence, the last ones first: late tokens see most
    const int pairs = a.c.n_kv * a.parts, x = (int)blockIdx.x / pairs, pair = (int)blockIdx.x % pairs;
    const int share = (a.tile_blocks + a.n_seq - 1) / a.n_seq, block = (x % a.n_seq) * share + share - 1 - x / a.n_seq;
    if (block >= a.tile_blocks) return;
    const int lane = threadIdx.x & 63;
    int b = -1;
    for (int b0 = 0; b0 < a.n_seq; b0 += 64) {
        const int i = min(b0 + lane, a.n_seq - 1);
        const int64_t first = (int64_t)min(max(a.starts[i], 0), a.n_tok) * a.group / ROWS + i;
        const int n = __popcll(__ballot(b0 + lane < a.n_seq && first <= block));
        b += n;
        if (n < 64) break;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b < 0) return;
    const Seq s = seq_of(a, b);
    const int64_t row0 = (block - ((int64_t)s.start * a.group / ROWS + b)) * ROWS;
    if (row0 >= s.rows || s.rows <= a.short_rows) return;
    many<F32, NG, SPARE, QUICK>(a, M, s, pair % a.c.n_kv, (int)row0, pair / a.c.n_kv);
}

// Workgroups [0, tile_wgs): blocks of 128 rows, gone through as MODE says; the others: a short sequence each.  QUICK: how a cap's tanh is
// computed.
template <bool F32, PgMode MODE, bool QUICK = !F32>
__global__ __launch_bounds__(MODE == PG_TWO_GROUPS ? 512 : 256, MODE == PG_SHORT && W <= 128 && W * kParts<F32> <= 256 ? 2 : 1) void k_attn_paged(const AttnPgArgs a)
{
    constexpr int NG = MODE == PG_TWO_GROUPS ? 2 : 1, NW = 4 * NG;
    union Mem {
        Many<NG> many;
        Few<NW> few;
    };
    __shared__ __align__(1024) char mem[MODE != PG_SHORT ? sizeof(Mem) : sizeof(Few<NW>)];
    Mem &M = *(Mem *)mem;
    if constexpr (MODE != PG_SHORT) {
        if ((int)blockIdx.x < a.tile_wgs) {
            many_rows<F32, NG, MODE == PG_SPARE, QUICK>(a, M.many);
            return;
        }
    }
    // (KV heads fastest: one's pages are read through one XCD's L2 where there are eight)
    const int i = blockIdx.x - a.tile_wgs, head = i % a.c.n_kv, rest = i / a.c.n_kv;
    const bool ranked = MODE == PG_SHORT && a.ranked;
    const int b = ranked ? nth_longest(a, rest / a.parts) : rest % a.n_seq, part = ranked ? rest % a.parts : rest / a.n_seq;
    const Seq s = seq_of(a, b);
    if (s.rows <= 0 || s.rows > kPgRows) return;
    few<F32, NW, QUICK>(a, M.few, s, head, part);
}

// Whether two groups of four waves find registers: 256 a lane.
template <bool F32> constexpr bool kTwoGroups = W <= 128 && W * (1 + kParts<F32>) <= (kParts<F32> == 1 ? 256 : 192);
// Whether PG_SPARE leaves room for three waves on a SIMD, where PG_ONE_GROUP has two.
template <bool F32> constexpr bool kSpare = W * kParts<F32> <= 64;

template <bool F32>
hipError_t launch(const AttnPgArgs &a, const AttnPgPlan &p, hipStream_t s)
{
    const unsigned n = (unsigned)p.blocks;
    if constexpr (!F32) {
        // (a large cap is rare: one group of waves on every block, so that the other instances need not hold its tanh as well, which
        // takes registers of theirs: mixed chunks and decodes with a window 41 us for 38)
        if (a.cap_in != 0.0f && a.cap_out > kQuickCap) {
            if (p.mode == PG_SHORT) k_attn_paged<F32, PG_SHORT, false><<<n, 256, 0, s>>>(a);
            else k_attn_paged<F32, PG_ONE_GROUP, false><<<n, 256, 0, s>>>(a);
            return hipGetLastError();
        }
    }
    if (p.mode == PG_SHORT) k_attn_paged<F32, PG_SHORT><<<n, 256, 0, s>>>(a);
    if (p.mode == PG_ONE_GROUP) k_attn_paged<F32, PG_ONE_GROUP><<<n, 256, 0, s>>>(a);
    if constexpr (kTwoGroups<F32>)
        if (p.mode == PG_TWO_GROUPS) k_attn_paged<F32, PG_TWO_GROUPS><<<n, 512, 0, s>>>(a);
    if constexpr (kSpare<F32>)
        if (p.mode == PG_SPARE) k_attn_paged<F32, PG_SPARE><<<n, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

#define SMX_PG_NAME_(f, w, b) f##_w##w##_b##b
#define SMX_PG_NAME(f, w, b) SMX_PG_NAME_(f, w, b)
hipError_t SMX_PG_NAME(launch_attn_paged, SMX_PG_W, SMX_PG_BF16)(const AttnPgArgs &a, const AttnPgPlan &p, hipStream_t s)
{
    return a.io == PG_F32 ? launch<true>(a, p, s) : launch<false>(a, p, s);
}
bool SMX_PG_NAME(attn_paged_has, SMX_PG_W, SMX_PG_BF16)(int io, PgMode m)
{
    return m == PG_TWO_GROUPS ? (io == PG_F32 ? kTwoGroups<true> : kTwoGroups<false>) : m != PG_SPARE || (io == PG_F32 ? kSpare<true> : kSpare<false>);
}

}  // namespace smx
