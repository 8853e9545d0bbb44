// k_kvcache.hip -- writing rows into the 8-bit KV cache and reading them back.
//
// A row x (head_dim values of one token's K or V in one KV head) is kept as Q8Tensor.Quantize keeps a
// block (Q8Tensor.cs:72-128): scale = fl32(max |x_i| / 127), code_i = the integer nearest to
// x_i / scale, ties to even, at most 127 in size.  The nearest integer is exact: a first guess n from
// the rounded quotient is at most one off, r = x - n scale is exact in fp32 (n scale and x agree in their
// leading bits, or n = 0), and 2 |r| against scale says which side of the border x lies on.  A row
// with a NaN or an infinity gets the scale NaN and zero codes: it reads back as NaN, and attention
// that sees it gives NaN.
//
// One workgroup handles 64 tokens of K or V of one KV head; 16 lanes share a row, so a row's maximum is four
// DPP steps.  K rows go straight to the cache.  V lies transposed, a byte per position: rows pass
// through LDS, and wherever four tokens follow one another from a position that is a multiple of 4
// (prompts) their bytes move as one dword; the rest (one token of each of many sequences) as bytes.
#include "smx_device.h"
#include "smx_internal.h"
#include "smx_kvcache.h"

namespace smx {

namespace {

constexpr int kT = 256;
constexpr int kRows = 64;   // tokens per workgroup

// Maximum of the 16 lanes of a row group.
__device__ __forceinline__ uint32_t row16_umax(uint32_t v)
{
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
    return v;
}

// The integer nearest to x / scale, ties to even, as a float; the integer n is at most one off.
__device__ __forceinline__ float nearest_code(float x, float scale, float n)
{
    const float r = 2.0f * __builtin_fmaf(-n, scale, x);
    const bool odd = ((int)n & 1) != 0;
    if (r > scale || (r == scale && odd)) n += 1.0f;
    else if (r < -scale || (r == -scale && odd)) n -= 1.0f;
    return fminf(127.0f, fmaxf(-127.0f, n));
}

// The places of a workgroup's 64 tokens, and how their V bytes move: row r stands for itself (one
// byte per dim), leads four rows (a dword), or is one of those three that follow.
struct Places {
    int slot[kRows], pos[kRows];   // slot < 0: no place
    int jobs[kRows];               // rows that move bytes; bit 8: four of them
    int n_jobs;
};

__device__ __forceinline__ void find_places(Places &S, const KvView &c, const int32_t *slots, const int32_t *pos, int t0,
                                            int n_tok)
{
    const int tid = threadIdx.x;
    if (tid < kRows) {
        int s = -1, p = 0;
        if (t0 + tid < n_tok) {
            s = slots[t0 + tid];
            p = pos[t0 + tid];
            if ((unsigned)s >= (unsigned)c.n_slots || (unsigned)p >= (unsigned)c.ctx) s = -1;
        }
        if (s < 0) p = 0;
        S.slot[tid] = s;
        S.pos[tid] = p;
        bool lead = s >= 0 && (p & 3) == 0 && tid + 3 < kRows;
#pragma unroll
        for (int k = 1; k < 4; k++) {
            const int so = __shfl_down(s, k, 64), po = __shfl_down(p, k, 64);
            lead = lead && so == s && po == p + k;
        }
        const uint64_t leads = __ballot(lead);
        // a row is taken along by a leader among the three rows before it: two leaders are at least
        // four rows apart, since both their positions are multiples of 4
        const bool follows = ((leads << 1 | leads << 2 | leads << 3) >> tid & 1) != 0;
        const bool job = s >= 0 && !follows;
        const uint64_t all = __ballot(job);
        if (job) S.jobs[__popcll(all & ((1ull << tid) - 1))] = tid | (lead ? 256 : 0);
        if (tid == 0) S.n_jobs = __popcll(all);
    }
    __syncthreads();
}

// W: the cache's row width (head_dim rounded up); VEC: rows may be read as float4.
template <int W, bool VEC>
__global__ __launch_bounds__(kT) void k_kv_append(KvView c, const float *__restrict__ k, int64_t k_stride,
                                                  const float *__restrict__ v, int64_t v_stride,
                                                  const int32_t *__restrict__ slots, const int32_t *__restrict__ pos,
                                                  int n_tok)
{
    constexpr int Q = (W + 63) / 64;   // groups of four values per lane
    __shared__ Places S;
    __shared__ uint32_t codes[kRows * (W / 4 + 1)];
    const int tid = threadIdx.x, lane16 = tid & 15;
    const int head = (blockIdx.x >> 1) % c.n_kv, t0 = (int)((blockIdx.x >> 1) / c.n_kv) * kRows;
    const bool is_v = blockIdx.x & 1;
    const float *src = is_v ? v : k;
    const int64_t stride = is_v ? v_stride : k_stride;
    const int n = min(kRows, n_tok - t0);

    float x[4][Q][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = (tid >> 4) + 16 * j;
        const float *p = src + (int64_t)(t0 + r) * stride + (int64_t)head * c.hd;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int d = 64 * q + 4 * lane16;
            if constexpr (VEC) {
                float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (r < n && d < c.hd) f = *(const float4 *)(p + d);
                x[j][q][0] = f.x, x[j][q][1] = f.y, x[j][q][2] = f.z, x[j][q][3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) x[j][q][e] = r < n && d + e < c.hd ? p[d + e] : 0.0f;
            }
        }
    }
    find_places(S, c, slots, pos, t0, n_tok);

#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = (tid >> 4) + 16 * j;
        uint32_t m = 0;
#pragma unroll
        for (int q = 0; q < Q; q++)
#pragma unroll
            for (int e = 0; e < 4; e++) m = max(m, __float_as_uint(x[j][q][e]) & 0x7FFFFFFFu);
        m = row16_umax(m);
        const bool finite = m < 0x7F800000u;
        const float scale = finite ? __uint_as_float(m) / 127.0f : __uint_as_float(0x7FC00000u);
        const int slot = S.slot[r], ps = S.pos[r];
        uint8_t *rec = c.base + c.tile_off(max(slot, 0), head, ps / kKvTile);
        // below 2^-100 the reciprocal could leave the range of fp32: divide
        const bool small = !(scale >= 7.8886090522101181e-31f);
        const float inv = small ? 0.0f : 1.0f / scale;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int d = 64 * q + 4 * lane16;
            uint32_t w = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float xe = x[j][q][e];
                float code = 0.0f;
                if (!small) {
                    code = nearest_code(xe, scale, __builtin_rintf(xe * inv));
                } else if (finite && scale > 0.0f) {
                    // (a subnormal scale may be far below max |x| / 127: clamped before the division)
                    const float xc = fminf(127.0f * scale, fmaxf(-127.0f * scale, xe));
                    code = nearest_code(xc, scale, __builtin_rintf(xc / scale));
                }
                w |= (uint32_t)((int)code + kKvZero) << (8 * e);
            }
            if (W % 64 == 0 || d < W) {
                if (is_v) codes[r * (W / 4 + 1) + d / 4] = w;
                else if (slot >= 0) *(uint32_t *)(rec + (size_t)(ps % kKvTile) * W + d) = w;
            }
        }
        if (slot >= 0 && lane16 == 0)
            ((float *)(rec + (size_t)2 * kKvTile * W))[(is_v ? kKvTile : 0) + ps % kKvTile] = scale;
    }
    if (!is_v) return;
    __syncthreads();
    const uint8_t *b = (const uint8_t *)codes;
    constexpr int RB = W + 4;   // bytes of a row in LDS
    const int jobs = S.n_jobs;
    for (int i = tid; i < jobs * W; i += kT) {
        const int d = i / jobs, jb = S.jobs[i - d * jobs], r = jb & 255;
        const int ps = S.pos[r];
        uint8_t *dst = c.base + c.tile_off(S.slot[r], head, ps / kKvTile) + (size_t)kKvTile * W + d * kKvTile +
                       kv_v_byte(ps % kKvTile);
        const uint8_t *s = b + r * RB + d;
        if (jb & 256) *(uint32_t *)dst = (uint32_t)s[0] | (uint32_t)s[RB] << 8 | (uint32_t)s[2 * RB] << 16 | (uint32_t)s[3 * RB] << 24;
        else *dst = s[0];
    }
}

// The values of one K or V row group of 64 tokens: rows of [n_tok][n_kv][hd]; tokens without a place give 0.
template <int W, bool VEC>
__global__ __launch_bounds__(kT) void k_kv_read(KvView c, const int32_t *__restrict__ slots,
                                                const int32_t *__restrict__ pos, int n_tok, float *__restrict__ k,
                                                float *__restrict__ v)
{
    constexpr int Q = (W + 63) / 64;
    __shared__ Places S;
    __shared__ uint32_t codes[kRows * (W / 4 + 1)];
    const int tid = threadIdx.x, lane16 = tid & 15;
    const int head = (blockIdx.x >> 1) % c.n_kv, t0 = (int)((blockIdx.x >> 1) / c.n_kv) * kRows;
    const bool is_v = blockIdx.x & 1;
    float *dst = is_v ? v : k;
    const int n = min(kRows, n_tok - t0);
    find_places(S, c, slots, pos, t0, n_tok);
    if (is_v) {
        uint8_t *b = (uint8_t *)codes;
        constexpr int RB = W + 4;
        const int jobs = S.n_jobs;
        for (int i = tid; i < jobs * W; i += kT) {
            const int d = i / jobs, jb = S.jobs[i - d * jobs], r = jb & 255;
            const int ps = S.pos[r];
            const uint8_t *s = c.base + c.tile_off(S.slot[r], head, ps / kKvTile) + (size_t)kKvTile * W + d * kKvTile +
                               kv_v_byte(ps % kKvTile);
            uint8_t *o = b + r * RB + d;
            if (jb & 256) {
                const uint32_t w = *(const uint32_t *)s;
                o[0] = (uint8_t)w, o[RB] = (uint8_t)(w >> 8), o[2 * RB] = (uint8_t)(w >> 16), o[3 * RB] = (uint8_t)(w >> 24);
            } else {
                o[0] = *s;
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = (tid >> 4) + 16 * j;
        if (r >= n) continue;
        const int slot = S.slot[r], ps = S.pos[r];
        const uint8_t *rec = c.base + c.tile_off(max(slot, 0), head, slot < 0 ? 0 : ps / kKvTile);
        const float scale = slot < 0 ? 0.0f : ((const float *)(rec + (size_t)2 * kKvTile * W))[(is_v ? kKvTile : 0) + ps % kKvTile];
        float *p = dst + ((int64_t)(t0 + r) * c.n_kv + head) * c.hd;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int d = 64 * q + 4 * lane16;
            if (d >= c.hd) continue;
            uint32_t w = 0x01010101u * kKvZero;
            if (slot >= 0) w = is_v ? codes[r * (W / 4 + 1) + d / 4] : *(const uint32_t *)(rec + (size_t)(ps % kKvTile) * W + d);
            float f[4];
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = (float)((int)(w >> (8 * e) & 255u) - kKvZero) * scale;
            if constexpr (VEC) {
                *(float4 *)(p + d) = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) p[d + e] = f[e];
            }
        }
    }
}

template <typename F>
hipError_t by_width(int w, F f)
{
    switch (w) {
    case 32: return f(std::integral_constant<int, 32>{});
    case 64: return f(std::integral_constant<int, 64>{});
    case 96: return f(std::integral_constant<int, 96>{});
    case 128: return f(std::integral_constant<int, 128>{});
    case 160: return f(std::integral_constant<int, 160>{});
    case 192: return f(std::integral_constant<int, 192>{});
    case 224: return f(std::integral_constant<int, 224>{});
    case 256: return f(std::integral_constant<int, 256>{});
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv_append(const KvView &c, const float *k, int64_t k_stride, const float *v, int64_t v_stride,
                            const int32_t *slots, const int32_t *pos, int n_tok, hipStream_t s)
{
    const unsigned blocks = (unsigned)((int64_t)((n_tok + kRows - 1) / kRows) * c.n_kv * 2);
    // float4 reads need 16-byte aligned rows (head_dim is a multiple of 8)
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && k_stride % 4 == 0 && v_stride % 4 == 0;
    return by_width(c.w, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (vec) k_kv_append<W, true><<<blocks, kT, 0, s>>>(c, k, k_stride, v, v_stride, slots, pos, n_tok);
        else k_kv_append<W, false><<<blocks, kT, 0, s>>>(c, k, k_stride, v, v_stride, slots, pos, n_tok);
        return hipGetLastError();
    });
}

hipError_t launch_kv_read(const KvView &c, const int32_t *slots, const int32_t *pos, int n_tok, float *k, float *v,
                          hipStream_t s)
{
    const unsigned blocks = (unsigned)((int64_t)((n_tok + kRows - 1) / kRows) * c.n_kv * 2);
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    return by_width(c.w, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (vec) k_kv_read<W, true><<<blocks, kT, 0, s>>>(c, slots, pos, n_tok, k, v);
        else k_kv_read<W, false><<<blocks, kT, 0, s>>>(c, slots, pos, n_tok, k, v);
        return hipGetLastError();
    });
}

}  // namespace smx
