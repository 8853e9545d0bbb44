// k_attn_paged_join.hip -- how the attention over the paged KV cache and the sum of received weights are cut up, their
// dispatch by row width and element type, and the sums of their parts.
#include <math.h>

#include <algorithm>

#include "smx_attn_paged.h"
#include "smx_device.h"
#include "smx_internal.h"

namespace smx {

namespace {

// out = sum_s 2^(e_s - E) acc_s / sum_s 2^(e_s - E) l_s over the parts s that have weight, E their largest exponent e.
struct Joined {
    float4 o;
    float l, top;
};

__device__ __forceinline__ void join(Joined &a, float4 v, float l, float e)
{
    if (e == -__builtin_huge_valf()) return;   // a part without weight may hold anything in v
    const float up = fmaxf(a.top, e);
    const float f = __builtin_amdgcn_exp2f(e - up), g = a.top == -__builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(a.top - up);
    a.top = up;
    a.l = a.l * g + l * f;
    a.o.x = a.o.x * g + v.x * f, a.o.y = a.o.y * g + v.y * f;
    a.o.z = a.o.z * g + v.z * f, a.o.w = a.o.w * g + v.w * f;
}

// What bounds it is the latency of the parts' loads: a thread takes four dims of every PP-th part of a row, requested
// four at a time, and PP threads join theirs through LDS in a fixed order.  Rows outside the sequences stay as they are.
template <int PP>
__global__ __launch_bounds__(256) void k_attn_paged_join(const AttnPgArgs a)
{
    constexpr int R = 256 / PP;   // threads of a block that each have other outputs
    __shared__ Joined S[PP > 1 ? PP - 1 : 1][PP > 1 ? R : 1];
    const int lane = threadIdx.x % R, pp = threadIdx.x / R;
    const int64_t i = (int64_t)blockIdx.x * R + lane, n_rows = (int64_t)a.n_tok * a.n_head;
    const int per = a.c.hd / 4;
    bool in = i < n_rows * per;
    const int64_t row = in ? i / per : 0;
    const int d = in ? 4 * (int)(i - row * per) : 0, token = (int)(row / a.n_head);
    in = in && token >= ld_uniform(a.starts) && token < ld_uniform(a.starts + a.n_seq);
    Joined J{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f, -__builtin_huge_valf()};
    for (int s0 = pp; s0 < a.parts; s0 += 4 * PP) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) ml[k] = *(const float2 *)(a.part_ml + (min(s0 + k * PP, a.parts - 1) * n_rows + row) * 2);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int s = min(s0 + k * PP, a.parts - 1);
            v[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (ml[k].x != -__builtin_huge_valf()) v[k] = *(const float4 *)(a.part_acc + (s * n_rows + row) * a.c.hd + d);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (s0 + k * PP < a.parts) join(J, v[k], ml[k].y, ml[k].x);
    }
    if constexpr (PP > 1) {
        if (pp > 0) S[pp - 1][lane] = J;
        __syncthreads();
        if (pp > 0) return;
#pragma unroll
        for (int k = 0; k < PP - 1; k++) {
            const Joined &T = S[k][lane];
            join(J, T.o, T.l, T.top);
        }
    }
    if (!in) return;
    const bool none = J.top == -__builtin_huge_valf();
    const float inv = none ? 0.0f : 1.0f / J.l;
    if (a.lse && d == 0) a.lse[row] = none ? J.top : (__builtin_amdgcn_logf(J.l) + J.top) * 0.69314718055994531f;
    const float o[4] = {J.o.x * inv, J.o.y * inv, J.o.z * inv, J.o.w * inv};
    const int64_t at = row * a.c.hd + d;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        if (a.io == PG_F32) ((float *)a.out)[at + e] = o[e];
        else if (a.io == PG_F16) ((_Float16 *)a.out)[at + e] = (_Float16)o[e];
        else ((__bf16 *)a.out)[at + e] = (__bf16)o[e];
    }
}

// The parts of received weights, and what there was before.
__global__ __launch_bounds__(256) void k_attn_mass_join(const AttnPgArgs a)
{
    const int64_t n = (int64_t)a.n_seq * a.c.n_kv * a.max_len, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t pair = i / a.max_len;
    const int p = (int)(i - pair * a.max_len);
    float sum = 0.0f;
    for (int k = 0; k < a.mass_parts; k++) sum += a.mass_part[k * n + i];
    const float was = a.mass && p < a.mass_width ? a.mass[pair * a.mass_stride + p] : 0.0f;
    a.mass_out[i] = p < a.lens[pair / a.c.n_kv] ? was + sum : 0.0f;
}

}  // namespace

#define SMX_ALL(X) X(32, 0) X(64, 0) X(96, 0) X(128, 0) X(192, 0) X(256, 0) X(32, 1) X(64, 1) X(96, 1) X(128, 1) X(192, 1) X(256, 1)
#define SMX_DECL(w, b)                                                                                      \
    hipError_t launch_attn_paged_w##w##_b##b(const AttnPgArgs &a, const AttnPgPlan &p, hipStream_t s);      \
    hipError_t launch_attn_mass_w##w##_b##b(const AttnPgArgs &a, const MassPgPlan &p, hipStream_t s);       \
    bool attn_paged_has_w##w##_b##b(int io, PgMode m);
SMX_ALL(SMX_DECL)
#undef SMX_DECL

AttnPgPlan attn_paged_plan(const PgView &c, int io, int n_tok, int n_head, int n_seq, int max_q, int max_len, int window)
{
    AttnPgPlan p{};
    const int64_t group = n_head / c.n_kv, rows = max_q * group;
    const int64_t tiles = std::max(1, (max_len + kPgTile - 1) / kPgTile);
    bool two = false, spare = false;
#define SMX_CASE(w_, b) if (c.w == w_ && c.bf16 == b) two = attn_paged_has_w##w_##_b##b(io, PG_TWO_GROUPS), spare = attn_paged_has_w##w_##_b##b(io, PG_SPARE);
    SMX_ALL(SMX_CASE)
#undef SMX_CASE
    constexpr int block = 4 * kPgRows;
    p.mode = rows <= kPgRows ? PG_SHORT : PG_ONE_GROUP;
    // what a block goes through at most, where the window says so, and how many blocks that is done by
    const int64_t span = window > 0 ? std::min<int64_t>(tiles, (window + (p.mode != PG_SHORT ? block / group + 1 : (int64_t)max_q)) / kPgTile + 2) : tiles;
    int64_t units = (int64_t)n_seq * c.n_kv, n = 1;
    p.chunk = p.mode != PG_SHORT ? 1 : 4;
    if (p.mode == PG_SHORT) {
        // Two workgroups for every compute unit, of four tiles at least, or two where that leaves most of the chip idle; up to
        // eight for long contexts while 32 tiles are left for each, the longest sequences' first, so that all end together (8
        // heads of 128 dims, 64 sequences of 2048 to 8192: 241 us for 252 in their own order and 260 in one part, 32 of 8000 to
        // 32768: 417 for 442 and 493; 64 of 8192: 376 for 367 in one part); but one part, which needs no second launch, up to 1024
        // positions of 64 dims or 512 of 128 (700 of 64, 4 heads: 10.7 us for 6.9 + 4.2 in six parts, and 4 us less for the
        // host to do).
        n = std::min((512 + units - 1) / units, (span + 3) / 4);
        if (n * units < 128) n = std::max(n, std::min((128 + units - 1) / units, (span + 1) / 2)), p.chunk = 2;
        n = std::max(n, std::min((2048 + units - 1) / units, span / 32));
        if (span * c.w <= 1024) n = 1;
    } else {
        p.tile_blocks = (int)(n_tok * group / block + n_seq);
        units = std::max<int64_t>(1, (n_tok * group + block - 1) / block) * c.n_kv;
        // Two groups of four waves on a block, which then has a compute unit to itself, while there is one for every block (1024
        // tokens over 1024 positions, 32 x 128 dims, 256 blocks: 27.8 us for 31.8 with one group); above that, where the
        // blocks that must wait can start early enough to end with the longest one.  Longest first, the 257th waits for the 256th, about
        // as long as itself; a block costs some six tiles beside its own (1536 over 1536, 384 blocks: 38.7 us for 43.6;
        // but 1280 over 4096, 320 blocks: 128 for 115, and 6 x 256 over 512, 384 blocks: 31 for 22).
        const double longest = span + 6.0, shortest = std::min<double>(span, (max_len - std::min(max_q, max_len)) / kPgTile) + 6.0;
        const double wgs = (double)((p.tile_blocks + n_seq - 1) / n_seq * (int64_t)n_seq * c.n_kv);   // (those that find no rows among them)
        if (two && (units <= 256 || 2 * (longest - (longest - shortest) * 256 / wgs) <= longest)) p.mode = PG_TWO_GROUPS;
        // More than two blocks for every compute unit: three at a time where their registers allow it (64 dims, 16 prompts of 1023,
        // 12 heads: 61 us for 71; 4096 over 4096, 32 heads over 8: 99 for 111; but 2048 over 8192, 512 blocks: 182 for 175).
        if (spare && units > 512) p.mode = PG_SPARE;
        // Parts up to one workgroup for every compute unit, of no fewer than four tiles.  n parts save 1 - 1 / n of the tiles'
        // time, about a microsecond each at 128 dims, and cost a launch, 4 us, and their sums' way to memory and back, 8 bytes
        // each at 5 TB/s: the best n is where these are equal, if that gains anything (64 tokens over 32768 positions, 16
        // blocks: 504 us in one part, 55 in 16; 512 over 4096, 128 blocks of fp32, 64 dims: 73 and 52 in two; two chunks of 512
        // with a window of 1024, 128 blocks of 128 dims: 40 and 58 in two).
        const double save = (double)span * c.w / 128, part = (double)n_tok * n_head * c.hd * 8 / 5e6;
        n = std::min({(int64_t)sqrt(save / part), 256 / units, (span + 3) / 4});
        if (n > 1 && save * (1 - 1.0 / n) < 4 + part * n) n = 1;
    }
    p.parts = (int)std::max<int64_t>(n, 1);
    const int64_t shares = p.mode != PG_SHORT ? (p.tile_blocks + n_seq - 1) / n_seq * (int64_t)n_seq : 0;   // (blocks in equal shares)
    p.tile_wgs = shares * c.n_kv * p.parts;
    // short sequences of a batch with longer ones go their own way
    p.blocks = p.tile_wgs + (p.mode == PG_SHORT || n_seq > 1 ? (int64_t)n_seq * c.n_kv * p.parts : 0);
    // (up to 512 workgroups all start at once)
    p.ranked = p.mode == PG_SHORT && n_seq > 1 && p.blocks > 512;
    p.work_bytes = p.parts > 1 ? (int64_t)p.parts * n_tok * n_head * (c.hd + 2) * 4 : 0;
    return p;
}

hipError_t launch_attn_paged(AttnPgArgs a, const AttnPgPlan &p, void *work, hipStream_t s)
{
    a.tile_wgs = (int)p.tile_wgs;
    a.tile_blocks = p.tile_blocks;
    a.short_rows = p.mode != PG_SHORT && a.n_seq > 1 ? kPgRows : 0;
    a.chunk = p.chunk;
    a.ranked = p.ranked;
    a.parts = p.parts;
    const int64_t rows = (int64_t)a.n_tok * a.n_head;
    a.part_acc = (float *)work;
    a.part_ml = work ? (float *)work + p.parts * rows * a.c.hd : nullptr;
    hipError_t e = hipErrorInvalidValue;
#define SMX_CASE(w_, b) if (a.c.w == w_ && a.c.bf16 == b) e = launch_attn_paged_w##w_##_b##b(a, p, s);
    SMX_ALL(SMX_CASE)
#undef SMX_CASE
    if (e != hipSuccess || p.parts == 1) return e;
    // about four parts per thread
    const int64_t n = rows * (a.c.hd / 4);
    if (p.parts <= 4) k_attn_paged_join<1><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    else if (p.parts <= 16) k_attn_paged_join<4><<<(unsigned)((n + 63) / 64), 256, 0, s>>>(a);
    else k_attn_paged_join<16><<<(unsigned)((n + 15) / 16), 256, 0, s>>>(a);
    return hipGetLastError();
}

// Parts of a query's values in k_attn_mass, and row blocks that it lays out at a time.
static int attn_mass_parts(const PgView &c, int io) { return io != PG_F32 ? 1 : c.bf16 ? 3 : 2; }
static int attn_mass_blocks(const PgView &c, int io)
{
    const int wide = attn_mass_parts(c, io) * c.w;
    return wide <= 256 ? 4 : wide <= 512 ? 2 : 1;
}

MassPgPlan attn_mass_plan(const PgView &c, int io, int n_head, int n_seq, int max_q, int max_len)
{
    MassPgPlan p{};
    // (max_q is a bound, and may be any: no call has rows of more than 2^31 - 1 values in all)
    const int64_t rows = std::min<int64_t>((int64_t)max_q * (n_head / c.n_kv), 0x7FFFFFFF / (c.n_kv * c.hd)), pairs = (int64_t)n_seq * c.n_kv;
    p.parts = 1;
    p.few = rows <= kPgRows;
    if (p.few) {
        // positions of a pair over enough workgroups for two on each compute unit, 128 at a time; over twice as many, the longest
        // sequences' first, where 2048 positions are left for each (8 heads of 128 dims, 64 sequences of 2048 to 8192: 145 us
        // for 162, 32 of 8000 to 32768: 263 for 320; 64 of 8192: 220 for 215; 16 of 8192 would take 48 for 43)
        const int64_t shares = std::max<int64_t>(std::min<int64_t>((1024 + pairs - 1) / pairs, max_len / 2048),
                                                 std::min<int64_t>((512 + pairs - 1) / pairs, (max_len + 127) / 128));
        p.blocks = pairs * std::max<int64_t>(1, shares);
        p.ranked = n_seq > 1 && p.blocks > 512;
        return p;
    }
    const int64_t keys = c.w <= 128 ? 256 : 128, units = pairs * ((max_len + keys - 1) / keys);
    const int nb = attn_mass_blocks(c, io);
    const int64_t blocks = (rows + 32 * nb - 1) / (32 * nb);
    // Rows of a part: as many as make two workgroups for every compute unit, but 256 at least at 128 dims, which with
    // the sum of parts take 10 us (512 tokens over 512 positions, 32 heads over 8 of 128: 43 us in parts of 1024, 21 of 256; 512 over 4096:
    // 44, 32 of 512 and 35 of 256); 1024 are enough, so that early positions, which more rows see, do not end last (4095
    // tokens: 130 us, 140 in parts of 2048, 358 in one); but no more parts than make 3000 workgroups, whose work memory
    // is at most 6 MB or so (2048 over 32768: 610 us with 3 parts, 632 with 8).
    const int64_t few = std::max<int64_t>(32768 / (c.w * attn_mass_parts(c, io)), (rows * units + 511) / 512);
    const int64_t many = std::max<int64_t>(1024, (rows * units + 2999) / 3000);
    p.per = (int)std::min((std::min(few, many) + 32 * nb - 1) / (32 * nb), blocks);
    p.parts = (int)((blocks + p.per - 1) / p.per);
    p.blocks = units * p.parts;
    p.work_bytes = p.parts > 1 ? (int64_t)p.parts * pairs * max_len * 4 : 0;
    return p;
}

hipError_t launch_attn_mass(AttnPgArgs a, const MassPgPlan &p, void *work, hipStream_t s)
{
    a.mass_parts = p.parts;
    a.mass_per = p.per;
    a.ranked = p.ranked;
    a.mass_part = (float *)work;
    hipError_t e = hipErrorInvalidValue;
#define SMX_CASE(w_, b) if (a.c.w == w_ && a.c.bf16 == b) e = launch_attn_mass_w##w_##_b##b(a, p, s);
    SMX_ALL(SMX_CASE)
#undef SMX_CASE
    if (e != hipSuccess || p.parts == 1) return e;
    const int64_t n = (int64_t)a.n_seq * a.c.n_kv * a.max_len;
    k_attn_mass_join<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
