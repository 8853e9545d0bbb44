// k_kvcache.hip -- writing rows into the 8-bit KV cache and reading them back.
//
// A row x (head_dim values of one token's K or V in one KV head) is kept as Q8Tensor.Quantize keeps a
// block (Q8Tensor.cs:72-128): scale = fl32(max |x_i| / 127), code_i = the integer nearest to
// x_i / scale, ties to even, at most 127 in size.  The nearest integer is exact.  x times the rounded
// reciprocal is within 2^-16 of x / scale, so its nearest integer n is the code unless it comes within
// 2^-15 of a half; lanes that hold such a value look again: r = x - n scale is exact in fp32 (n scale
// and x agree in their leading bits, or n = 0), and 2 |r| against scale says which side of the border x lies on.
// (Looking at every value that way took 18 instructions each, where memory leaves time for about ten.)  A row
// with a NaN or an infinity gets the scale NaN and zero codes: it reads back as NaN, and attention
// that sees it gives NaN.
//
// One workgroup handles 64 (or 16) tokens of K or V of one KV head; 16 lanes share a row, so a row's maximum is four
// DPP steps.  K rows go straight to the cache.  V lies transposed, a byte per position: rows pass
// through LDS, and wherever four tokens follow one another from a position that is a multiple of 4
// (prompts) their bytes move as 4 x 4 blocks, a dword for each dim; the rest (one token of each of many
// sequences) as bytes.  16 prompts of 2047 tokens, 8 heads of 128: writing 67 us (5.0 TB/s of floats and codes),
// reading 54; one token for each of 16 sequences, 4 heads of 64: 4.1 and 4.3, near an empty launch.
#include "smx_device.h"
#include "smx_internal.h"
#include "smx_kvcache.h"

namespace smx {

namespace {

constexpr int kT = 256;
constexpr int kRows = 64;   // tokens per workgroup, at most

typedef float float4v __attribute__((ext_vector_type(4)));

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

// Columns of a 4 x 4 block of bytes from its rows, and back.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4])
{
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u);
    w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// The places of a workgroup's 64 tokens, and how their V bytes move: in fours, by the row that leads them,
// or singly.
struct Places {
    int slot[kRows], pos[kRows];   // slot < 0: no place
    int four[kRows / 4], one[kRows];
    int n_four, n_one;
};

template <int ROWS>
__device__ __forceinline__ void find_places(Places &S, const KvView &c, const int32_t *slots, const int32_t *pos, int t0,
                                            int n_tok)
{
    const int tid = threadIdx.x;
    if (tid < ROWS) {
        int s = -1, p = 0;
        if (t0 + tid < n_tok) {
            s = slots[t0 + tid];
            p = pos[t0 + tid];
            if ((unsigned)s >= (unsigned)c.n_slots || (unsigned)p >= (unsigned)c.ctx) s = -1;
        }
        if (s < 0) p = 0;
        S.slot[tid] = s;
        S.pos[tid] = p;
        bool lead = s >= 0 && (p & 3) == 0 && tid + 3 < ROWS;
#pragma unroll
        for (int k = 1; k < 4; k++) {
            const int so = __shfl_down(s, k, 64), po = __shfl_down(p, k, 64);
            lead = lead && so == s && po == p + k;
        }
        // two leaders are at least four rows apart, since both their positions are multiples of 4
        const uint64_t leads = __ballot(lead);
        const bool led = ((leads | leads << 1 | leads << 2 | leads << 3) >> tid & 1) != 0;
        const uint64_t ones = __ballot(s >= 0 && !led);
        const uint64_t before = (1ull << tid) - 1;
        if (lead) S.four[__popcll(leads & before)] = tid;
        if (s >= 0 && !led) S.one[__popcll(ones & before)] = tid;
        if (tid == 0) S.n_four = __popcll(leads), S.n_one = __popcll(ones);
    }
    __syncthreads();
}

// f(four, 4-dim group) for all fours and f(one, dim) for all single rows, fours and rows fastest, so that
// neighbouring lanes have neighbouring positions of one dim.
template <int W, typename F4, typename F1>
__device__ __forceinline__ void each_place(const Places &S, F4 four, F1 one)
{
    const int n4 = S.n_four, n1 = S.n_one;
    // quotients of i < 2^14 by n <= 64
    const uint32_t m4 = 0xFFFFFFFFu / (uint32_t)max(n4, 1) + 1u, m1 = 0xFFFFFFFFu / (uint32_t)max(n1, 1) + 1u;
    for (int i = threadIdx.x; i < n4 * (W / 4); i += kT) {
        const int q = n4 == 1 ? i : (int)__umulhi((uint32_t)i, m4);
        four(S.four[i - q * n4], q);
    }
    for (int i = threadIdx.x; i < n1 * W; i += kT) {
        const int d = n1 == 1 ? i : (int)__umulhi((uint32_t)i, m1);
        one(S.one[i - d * n1], d);
    }
}

// W: the cache's row width (head_dim rounded up); VEC: rows may be read as float4; NT: past the caches; ROWS:
// tokens per workgroup.
template <int W, bool VEC, bool NT, int ROWS>
__global__ __launch_bounds__(kT) void k_kv_append(KvView c, const float *__restrict__ k, int64_t k_stride,
                                                  const float *__restrict__ v, int64_t v_stride,
                                                  const int32_t *__restrict__ slots, const int32_t *__restrict__ pos,
                                                  int n_tok)
{
    constexpr int Q = (W + 63) / 64;   // groups of four values per lane
    __shared__ Places S;
    __shared__ uint32_t codes[ROWS * (W / 4 + 1)];
    const int tid = threadIdx.x, lane16 = tid & 15;
    const int head = (blockIdx.x >> 1) % c.n_kv, t0 = (int)((blockIdx.x >> 1) / c.n_kv) * ROWS;
    const bool is_v = blockIdx.x & 1;
    const float *src = is_v ? v : k;
    const int64_t stride = is_v ? v_stride : k_stride;
    const int n = min(ROWS, n_tok - t0);

    float x[ROWS / 16][Q][4];
#pragma unroll
    for (int j = 0; j < ROWS / 16; j++) {
        const int r = (tid >> 4) + 16 * j;
        const float *p = src + (int64_t)(t0 + r) * stride + (int64_t)head * c.hd;
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int d = 64 * q + 4 * lane16;
            if constexpr (VEC) {
                float4v f = {0.0f, 0.0f, 0.0f, 0.0f};
                if (r < n && d < c.hd) f = NT ? __builtin_nontemporal_load((const float4v *)(p + d)) : *(const float4v *)(p + d);
#pragma unroll
                for (int e = 0; e < 4; e++) x[j][q][e] = f[e];
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) x[j][q][e] = r < n && d + e < c.hd ? p[d + e] : 0.0f;
            }
        }
    }
    find_places<ROWS>(S, c, slots, pos, t0, n_tok);

#pragma unroll
    for (int j = 0; j < ROWS / 16; j++) {
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
        // x inv + 1.5 2^23 + 128 has its nearest integer, plus 128, in the low byte
        constexpr float kMagic = 12582912.0f + kKvZero;
        float far = 0.0f;
        uint32_t w[Q];
#pragma unroll
        for (int q = 0; q < Q; q++) {
            uint32_t u[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float xe = x[j][q][e], f = __builtin_fmaf(xe, inv, kMagic);
                far = fmaxf(far, fabsf(__builtin_fmaf(xe, inv, kMagic - f)));
                u[e] = __float_as_uint(f);
            }
            w[q] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(u[1], u[0], 0x0C0C0400u), 0x05040100u);
        }
        if (small || !(far < 0.5f - 3.0517578125e-5f)) {   // (NaN: not finite)
#pragma unroll
            for (int q = 0; q < Q; q++) {
                w[q] = 0;
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
                    w[q] |= (uint32_t)((int)code + kKvZero) << (8 * e);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < Q; q++) {
            const int d = 64 * q + 4 * lane16;
            if (W % 64 == 0 || d < W) {
                if (is_v) codes[r * (W / 4 + 1) + d / 4] = w[q];
                else if (slot >= 0) *(uint32_t *)(rec + (size_t)(ps % kKvTile) * W + d) = w[q];
            }
        }
        if (slot >= 0 && lane16 == 0)
            ((float *)(rec + (size_t)2 * kKvTile * W))[(is_v ? kKvTile : 0) + ps % kKvTile] = scale;
    }
    if (!is_v) return;
    __syncthreads();
    constexpr int RD = W / 4 + 1;   // dwords of a row in LDS
    const auto place = [&](int r) {
        const int ps = S.pos[r];
        return c.base + c.tile_off(S.slot[r], head, ps / kKvTile) + (size_t)kKvTile * W + kv_v_byte(ps % kKvTile);
    };
    each_place<W>(
        S,
        [&](int r, int q) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = codes[(r + k) * RD + q];
            transpose4(w);
            uint8_t *dst = place(r) + 4 * q * kKvTile;
#pragma unroll
            for (int k = 0; k < 4; k++) *(uint32_t *)(dst + k * kKvTile) = w[k];
        },
        [&](int r, int d) { place(r)[d * kKvTile] = ((const uint8_t *)codes)[4 * r * RD + d]; });
}

// The values of K or V of a workgroup's tokens: rows of [n_tok][n_kv][hd]; tokens without a place give 0.
template <int W, bool VEC, bool NT, int ROWS>
__global__ __launch_bounds__(kT) void k_kv_read(KvView c, const int32_t *__restrict__ slots,
                                                const int32_t *__restrict__ pos, int n_tok, float *__restrict__ k,
                                                float *__restrict__ v)
{
    constexpr int Q = (W + 63) / 64;
    __shared__ Places S;
    __shared__ uint32_t codes[ROWS * (W / 4 + 1)];
    const int tid = threadIdx.x, lane16 = tid & 15;
    const int head = (blockIdx.x >> 1) % c.n_kv, t0 = (int)((blockIdx.x >> 1) / c.n_kv) * ROWS;
    const bool is_v = blockIdx.x & 1;
    float *dst = is_v ? v : k;
    const int n = min(ROWS, n_tok - t0);
    find_places<ROWS>(S, c, slots, pos, t0, n_tok);
    if (is_v) {
        constexpr int RD = W / 4 + 1;
        const auto place = [&](int r) {
            const int ps = S.pos[r];
            return c.base + c.tile_off(S.slot[r], head, ps / kKvTile) + (size_t)kKvTile * W + kv_v_byte(ps % kKvTile);
        };
        each_place<W>(
            S,
            [&](int r, int q) {
                const uint8_t *src = place(r) + 4 * q * kKvTile;
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] = *(const uint32_t *)(src + k * kKvTile);
                transpose4(w);
#pragma unroll
                for (int k = 0; k < 4; k++) codes[(r + k) * RD + q] = w[k];
            },
            [&](int r, int d) { ((uint8_t *)codes)[4 * r * RD + d] = place(r)[d * kKvTile]; });
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < ROWS / 16; j++) {
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
            float4v f;
#pragma unroll
            for (int e = 0; e < 4; e++) f[e] = (float)((int)(w >> (8 * e) & 255u) - kKvZero) * scale;
            if constexpr (NT) {
                __builtin_nontemporal_store(f, (float4v *)(p + d));
            } else if constexpr (VEC) {
                *(float4v *)(p + d) = f;
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

// Tokens per workgroup: 64, or 16 where that would leave compute units without work (a token for each of 128
// sequences, 8 heads of 128: writing 11.8 -> 6.9 us, reading 13.8 -> 5.9).
bool few(const KvView &c, int n_tok) { return (int64_t)((n_tok + kRows - 1) / kRows) * c.n_kv * 2 < 512; }

unsigned blocks_of(const KvView &c, int n_tok, int rows) { return (unsigned)((int64_t)((n_tok + rows - 1) / rows) * c.n_kv * 2); }

// Bytes of K and V as floats.
double float_bytes(const KvView &c, int n_tok) { return 8.0 * n_tok * c.n_kv * c.hd; }

}  // namespace

hipError_t launch_kv_append(const KvView &c, const float *k, int64_t k_stride, const float *v, int64_t v_stride,
                            const int32_t *slots, const int32_t *pos, int n_tok, hipStream_t s)
{
    const unsigned n64 = blocks_of(c, n_tok, 64), n16 = blocks_of(c, n_tok, 16);
    // float4 reads need 16-byte aligned rows (head_dim is a multiple of 8)
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && k_stride % 4 == 0 && v_stride % 4 == 0;
    // rows that the caches (8 x 4 MB) could not keep anyway: 16 x 2047 tokens of 8 x 128 dims 73 -> 69 us; 4 x 2000 of 1 x 256
    // (16 MB) 10.8 -> 11.1
    const bool nt = float_bytes(c, n_tok) > 32.0 * (1 << 20);
    return by_width(c.w, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (!vec) k_kv_append<W, false, false, 64><<<n64, kT, 0, s>>>(c, k, k_stride, v, v_stride, slots, pos, n_tok);
        else if (few(c, n_tok)) k_kv_append<W, true, false, 16><<<n16, kT, 0, s>>>(c, k, k_stride, v, v_stride, slots, pos, n_tok);
        else if (nt) k_kv_append<W, true, true, 64><<<n64, kT, 0, s>>>(c, k, k_stride, v, v_stride, slots, pos, n_tok);
        else k_kv_append<W, true, false, 64><<<n64, kT, 0, s>>>(c, k, k_stride, v, v_stride, slots, pos, n_tok);
        return hipGetLastError();
    });
}

hipError_t launch_kv_read(const KvView &c, const int32_t *slots, const int32_t *pos, int n_tok, float *k, float *v,
                          hipStream_t s)
{
    const unsigned n64 = blocks_of(c, n_tok, 64), n16 = blocks_of(c, n_tok, 16);
    const bool vec = (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    // from a few MB on, values written past the caches do not push the codes out of them: 16 x 2047 tokens of 8 x 128 dims
    // 86 -> 51 us, 4096 of 4 x 64 (8 MB) 6.2 -> 5.7; 16 of 4 x 64 4.5 -> 4.8
    const bool nt = float_bytes(c, n_tok) > 4.0 * (1 << 20);
    return by_width(c.w, [&](auto w) {
        constexpr int W = decltype(w)::value;
        if (!vec) k_kv_read<W, false, false, 64><<<n64, kT, 0, s>>>(c, slots, pos, n_tok, k, v);
        else if (few(c, n_tok)) k_kv_read<W, true, false, 16><<<n16, kT, 0, s>>>(c, slots, pos, n_tok, k, v);
        else if (nt) k_kv_read<W, true, true, 64><<<n64, kT, 0, s>>>(c, slots, pos, n_tok, k, v);
        else k_kv_read<W, true, false, 64><<<n64, kT, 0, s>>>(c, slots, pos, n_tok, k, v);
        return hipGetLastError();
    });
}

}  // namespace smx
