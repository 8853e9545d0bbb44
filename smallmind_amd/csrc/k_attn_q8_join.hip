// k_attn_q8_join.hip -- the plan of the attention over the 8-bit KV cache and the sum of its parts.
#include <math.h>

#include <algorithm>

#include "smx_attn_q8.h"
#include "smx_device.h"
#include "smx_internal.h"

namespace smx {

namespace {

// out = sum_s 2^(c (m_s - M)) acc_s / sum_s 2^(c (m_s - M)) l_s over the parts s that have weight, M their largest m.
// What bounds it is the latency of the parts' loads, so a thread takes four dims of every PP-th part of a row,
// requested four at a time, and PP threads join theirs through LDS in a fixed order.  Rows of a sequence
// without a slot are 0.
struct Joined {
    float4 o;
    float l, top;
};

__device__ __forceinline__ void join(Joined &a, float4 v, float l, float m, float c)
{
    if (l == 0.0f) return;   // a part without weight may hold anything in v
    const float up = fmaxf(a.top, m);
    // (-inf - -inf where nothing but NaN has been seen: the sum is NaN already)
    const float f = __builtin_amdgcn_exp2f((m - up) * c), g = a.l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f((a.top - up) * c);
    a.top = up;
    a.l = a.l * g + l * f;
    a.o.x = a.o.x * g + v.x * f, a.o.y = a.o.y * g + v.y * f;
    a.o.z = a.o.z * g + v.z * f, a.o.w = a.o.w * g + v.w * f;
}

template <int PP>
__global__ __launch_bounds__(256) void k_attn_q8_join(const AttnQ8Args a)
{
    constexpr int R = 256 / PP;   // threads of a block that each have other outputs
    __shared__ Joined S[PP > 1 ? PP - 1 : 1][PP > 1 ? R : 1];
    const int lane = threadIdx.x % R, pp = threadIdx.x / R;
    const int64_t i = (int64_t)blockIdx.x * R + lane;
    const int per = a.hd / 4;
    const bool in = i < a.n_rows * per;
    const int64_t row = in ? i / per : 0;
    const int d = in ? 4 * (int)(i - row * per) : 0;
    Joined J{make_float4(0.0f, 0.0f, 0.0f, 0.0f), 0.0f, -__builtin_huge_valf()};
    for (int s0 = pp; s0 < a.parts; s0 += 4 * PP) {
        float2 ml[4];
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int s = min(s0 + k * PP, a.parts - 1);
            ml[k] = *(const float2 *)(a.part_ml + (s * a.n_rows + row) * 2);
            v[k] = *(const float4 *)(a.part_acc + (s * a.n_rows + row) * a.hd + d);
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (s0 + k * PP < a.parts) join(J, v[k], ml[k].y, ml[k].x, a.scale_log2e);
    }
    if constexpr (PP > 1) {
        if (pp > 0) S[pp - 1][lane] = J;
        __syncthreads();
        if (pp > 0) return;
#pragma unroll
        for (int k = 0; k < PP - 1; k++) {
            const Joined &T = S[k][lane];
            join(J, T.o, T.l, T.top, a.scale_log2e);
        }
    }
    if (!in) return;
    const int seq = (int)(row / ((int64_t)a.n_q * a.n_head));
    const bool active = (unsigned)a.slots[seq] < (unsigned)a.n_slots;
    const float inv = !active || J.l == 0.0f ? 0.0f : 1.0f / J.l;
    if (!active) J.o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float *dst = a.out + row * a.hd + d;
    if (a.out_vec) {
        *(float4 *)dst = make_float4(J.o.x * inv, J.o.y * inv, J.o.z * inv, J.o.w * inv);
    } else {
        dst[0] = J.o.x * inv, dst[1] = J.o.y * inv, dst[2] = J.o.z * inv, dst[3] = J.o.w * inv;
    }
}

// Cuts a length into chunks, given the workgroups `units` that every chunk makes.  Two workgroups per compute unit
// (512) keep it busy; up to there chunks of at least four tiles, one for each wave, as a shorter one spends
// its time on the queries (64 sequences over 2048 shared positions, 128 dims: 23.5 us in chunks of four, 31 of
// two).  Where that leaves most of the chip idle, chunks of two tiles (1 x 1024, 128 dims: 9.4 for 9.7 us; 16 sequences
// over 512 shared positions: 10.1 for 11.6).
void cut(int len, int64_t units, int *chunk, int *splits)
{
    const int64_t tiles = (len + kKvTile - 1) / kKvTile;
    int64_t n = std::min((512 + units - 1) / units, (tiles + 3) / 4);
    if (n * units < 128) n = std::max(n, std::min((128 + units - 1) / units, (tiles + 1) / 2));
    n = std::max<int64_t>(n, 1);
    int64_t c = (tiles + n - 1) / n;
    if (c > 4) c = (c + 3) / 4 * 4;
    *chunk = (int)std::max<int64_t>(c, 1) * kKvTile;
    *splits = (len + *chunk - 1) / *chunk;
}

// A single part writes the outputs itself, unless it is the prefix, which knows no slots.
bool attn_q8_direct(const AttnQ8Plan &p) { return p.parts == 1 && p.own_splits == 1; }

}  // namespace

#define SMX_W(w) hipError_t launch_attn_q8_w##w(const AttnQ8Args &a, const AttnQ8Plan &p, hipStream_t s);
SMX_W(32) SMX_W(64) SMX_W(96) SMX_W(128) SMX_W(160) SMX_W(192) SMX_W(224) SMX_W(256)
#undef SMX_W

AttnQ8Plan attn_q8_plan(const KvView &c, int n_seq, int n_q, int n_head, int prefix_len, int max_len)
{
    AttnQ8Plan p{};
    const int64_t group = n_head / c.n_kv, own_rows = n_q * group, pre_rows = n_seq * own_rows;
    p.own_blocks = (int)((own_rows + 15) / 16);
    if (prefix_len > 0) {
        // several blocks of rows: the tiles are turned into fp16 once for four of them
        p.pre = pre_rows > 16 ? PRE_ROWS : PRE_STREAM;
        const int block = p.pre == PRE_ROWS ? 64 : 16;
        p.pre_blocks = (int)((pre_rows + block - 1) / block);
    }
    const int64_t own_units = (int64_t)n_seq * c.n_kv * p.own_blocks, pre_units = (int64_t)c.n_kv * p.pre_blocks;
    cut(max_len, own_units, &p.own_chunk, &p.own_splits);
    if (prefix_len > 0) {
        cut(prefix_len, pre_units, &p.pre_chunk, &p.pre_splits);
    } else if ((int64_t)(max_len + kKvTile - 1) / kKvTile * c.w <= 1024) {
        // a single part, which needs no second launch: 512 positions of 64 dims 6.3 us for 7.8 in two parts, 1024 8.6
        // for 7.9 and the launch saved, 512 of 128 dims 8.8 for 9.5, 512 of 256 dims 14 for 12
        p.own_chunk = std::max(1, (max_len + kKvTile - 1) / kKvTile) * kKvTile;
        p.own_splits = max_len > 0 ? 1 : 0;
    }
    // read once, and more than the memory-side cache holds from call to call (256 MB): 64 x 8192 positions of 8 x 128 dims
    // 139 -> 132 us; 32 x 2048 of them, which it holds, 24 -> 27
    p.past_caches = p.own_blocks == 1 && (double)n_seq * c.n_kv * max_len * 2 * c.w > 256.0 * (1 << 20);
    p.parts = p.own_splits + p.pre_splits;
    p.pre_wgs = pre_units * p.pre_splits;
    p.blocks = p.pre_wgs + own_units * p.own_splits;
    const int64_t rows = (int64_t)n_seq * n_q * n_head;
    p.work_bytes = attn_q8_direct(p) ? 0 : p.parts * rows * (int64_t)(c.hd + 2) * 4;
    return p;
}

hipError_t launch_attn_q8(const KvView &c, const AttnQ8Plan &p, const float *q, int64_t q_stride, float *out, int n_seq,
                          int n_q, int n_head, int prefix_slot, int prefix_len, const int32_t *slots, const int32_t *lens,
                          int max_len, void *work, hipStream_t s)
{
    AttnQ8Args a{};
    a.q = q;
    a.out = out;
    a.cache = c.base;
    a.head_bytes = (size_t)c.tiles * kv_tile_bytes(c.w);
    a.slots = slots;
    a.lens = lens;
    a.n_rows = (int64_t)n_seq * n_q * n_head;
    a.part_acc = (float *)work;
    a.part_ml = work ? (float *)work + p.parts * a.n_rows * c.hd : nullptr;
    a.q_stride = q_stride;
    a.inv_group = (double)c.n_kv / n_head;
    a.scale_log2e = (float)(1.4426950408889634 * 16.0 / sqrt((double)c.hd));
    a.q_vec = ((uintptr_t)q & 15) == 0 && q_stride % 4 == 0;
    a.out_vec = ((uintptr_t)out & 15) == 0;
    a.n_slots = c.n_slots;
    a.n_seq = n_seq;
    a.n_q = n_q;
    a.n_head = n_head;
    a.n_kv = c.n_kv;
    a.hd = c.hd;
    a.max_len = max_len;
    a.own_chunk = p.own_chunk;
    a.own_splits = p.own_splits;
    a.own_blocks = p.own_blocks;
    a.prefix_slot = prefix_slot;
    a.prefix_len = prefix_len;
    a.pre_chunk = p.pre_chunk;
    a.pre_splits = p.pre_splits;
    a.pre_wgs = (int)p.pre_wgs;
    a.parts = p.parts;
    a.direct = attn_q8_direct(p);
    if (p.blocks) {
        hipError_t e = hipErrorInvalidValue;
#define SMX_W(w) case w: e = launch_attn_q8_w##w(a, p, s); break;
        switch (c.w) { SMX_W(32) SMX_W(64) SMX_W(96) SMX_W(128) SMX_W(160) SMX_W(192) SMX_W(224) SMX_W(256) }
#undef SMX_W
        if (e != hipSuccess) return e;
    }
    if (a.direct) return hipSuccess;
    // about four parts per thread
    const int64_t n = a.n_rows * (c.hd / 4);
    if (p.parts <= 4) k_attn_q8_join<1><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a);
    else if (p.parts <= 16) k_attn_q8_join<4><<<(unsigned)((n + 63) / 64), 256, 0, s>>>(a);
    else k_attn_q8_join<16><<<(unsigned)((n + 15) / 16), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
