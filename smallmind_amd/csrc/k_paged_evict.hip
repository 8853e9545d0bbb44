// k_paged_evict.hip -- eviction from the paged KV cache: of every sequence and KV head the last n_recent positions and
// those others that have received the most weight, n_keep in all, copied in their order to other pages.
//
// Mathematics.  With n positions, r = min(n_recent, n_keep, n) of them the last, m = min(n, n_keep) - r of the first n - r are chosen:
// those whose weight is above the m-th largest, and of those equal to it the first.  The m-th largest is found digit
// by digit: weights as unsigned numbers of the same order, a count of each value of the leading 8 bits, and so on down
// the four bytes.  A NaN counts as less than every number, -0 as 0.
//
// Layout.  Choosing: one workgroup per (sequence, KV head); a thread owns SEG consecutive positions of each segment of
// 1024 * SEG, so that one scan over the threads gives every position its place in order.  Up to one segment the weights
// stay in registers through all passes; longer sequences read them again (from the L2).  Copying: a lane per
// 16-byte unit, rows anywhere in the pages.
#include "smx_device.h"
#include "smx_internal.h"

namespace smx {

namespace {

constexpr int kSeg = 16;                // positions of a thread
constexpr int kThreads = 1024;
constexpr int kSegment = kSeg * kThreads;

// Larger weights as larger numbers, none of them 0 but NaN's.
__device__ __forceinline__ uint32_t order_of(float f)
{
    const uint32_t u = __float_as_uint(f + 0.0f);   // (-0 becomes 0)
    if (f != f) return 0u;
    return (u >> 31) ? ~u : u | 0x80000000u;
}

struct Choose {
    uint32_t hist[16][256];   // a count for each wave: equal weights are common
    uint32_t total[256];
    uint32_t wave_gt[16], wave_eq[16];
    uint32_t digit, above, least;
};

__global__ __launch_bounds__(kThreads) void k_paged_choose(const PgEvictArgs a)
{
    __shared__ Choose S;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = blockIdx.x / a.c.n_kv, h = blockIdx.x - b * a.c.n_kv;
    const int n = min(max(a.lens[b], 0), a.max_len);
    const int keep = min(n, a.n_keep), recent = min(a.n_recent, keep), cand = n - recent;
    const uint32_t want = (uint32_t)(keep - recent);
    const float *mass = a.mass + (int64_t)blockIdx.x * a.mass_stride;
    int32_t *kept = a.kept + (int64_t)blockIdx.x * a.n_keep;
    float *out = a.new_mass + (int64_t)blockIdx.x * a.n_keep;
    if (h == 0 && tid == 0) a.new_lens[b] = keep;

    uint32_t key[kSeg];
    const auto load = [&](int s0) {
#pragma unroll
        for (int i = 0; i < kSeg; i++) {
            const int p = s0 + tid * kSeg + i;
            key[i] = p < cand ? order_of(mass[p]) : 0u;
        }
    };
    load(0);
    uint32_t least = 0, ties = 0;       // the m-th largest, and how many equal to it are kept
    const bool all = want >= (uint32_t)cand;
    if (want > 0 && !all) {
        uint32_t left = want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 16 * 256; i += kThreads) (&S.hist[0][0])[i] = 0;
            __syncthreads();
            for (int s0 = 0; s0 < cand; s0 += kSegment) {
                if (cand > kSegment) load(s0);
#pragma unroll
                for (int i = 0; i < kSeg; i++) {
                    const bool in = s0 + tid * kSeg + i < cand && (shift == 24 || (key[i] >> (shift + 8)) == (least >> (shift + 8)));
                    if (in) atomicAdd(&S.hist[wave][(key[i] >> shift) & 255u], 1u);
                }
            }
            __syncthreads();
            if (tid < 256) {
                uint32_t t = 0;
#pragma unroll
                for (int w = 0; w < 16; w++) t += S.hist[w][tid];
                S.total[tid] = t;
            }
            __syncthreads();
            // the largest digit with `left` or more at or above it
            if (wave == 0) {
                uint32_t c[4], sum = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) c[i] = S.total[4 * lane + i], sum += c[i];
                uint32_t above = sum;   // of this lane's digits and all higher ones
                for (int o = 1; o < 64; o <<= 1) {
                    const uint32_t v = __shfl_down(above, o, 64);
                    if (lane + o < 64) above += v;
                }
                above -= sum;
#pragma unroll
                for (int i = 3; i >= 0; i--) {
                    if (above < left && above + c[i] >= left) S.digit = 4 * lane + i, S.above = above;
                    above += c[i];
                }
            }
            __syncthreads();
            least |= S.digit << shift;
            left -= S.above;
            __syncthreads();
        }
        ties = left;
    }
    // in order of position: every one above `least`, and the first `ties` equal to it
    uint32_t eq_before = 0, at_before = 0;
    for (int s0 = 0; s0 < cand && want > 0; s0 += kSegment) {
        if (cand > kSegment) load(s0);
        uint32_t gt = 0, eq = 0;
#pragma unroll
        for (int i = 0; i < kSeg; i++) {
            const bool in = s0 + tid * kSeg + i < cand;
            gt += in && (all || key[i] > least);
            eq += in && !all && key[i] == least;
        }
        uint32_t g = gt, e = eq;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t x = __shfl_up(g, o, 64), y = __shfl_up(e, o, 64);
            if (lane >= o) g += x, e += y;
        }
        if (lane == 63) S.wave_gt[wave] = g, S.wave_eq[wave] = e;
        __syncthreads();
        uint32_t gb = g - gt, eb = e - eq, gall = 0, eall = 0;
#pragma unroll
        for (int w = 0; w < 16; w++) {
            if (w < wave) gb += S.wave_gt[w], eb += S.wave_eq[w];
            gall += S.wave_gt[w], eall += S.wave_eq[w];
        }
        eb += eq_before;
        uint32_t at = at_before + gb + min(eb, ties) - min(eq_before, ties);
#pragma unroll
        for (int i = 0; i < kSeg; i++) {
            const int p = s0 + tid * kSeg + i;
            if (p >= cand) continue;
            const bool is_eq = !all && key[i] == least;
            if (all || key[i] > least || (is_eq && eb < ties)) {
                kept[at] = p;
                out[at] = mass[p];
                at++;
            }
            eb += is_eq;
        }
        at_before += gall + min(eq_before + eall, ties) - min(eq_before, ties);
        eq_before += eall;
        __syncthreads();
    }
    for (int i = tid; i < recent; i += kThreads) {
        kept[want + i] = cand + i;
        out[want + i] = mass[cand + i];
    }
    for (int i = keep + tid; i < a.n_keep; i += kThreads) {
        kept[i] = -1;
        out[i] = 0.0f;
    }
}

// Rows kept[..] of the old pages to places 0 .. of the new ones.  blockIdx.y: (sequence, KV head).
__global__ __launch_bounds__(256) void k_paged_copy(const PgEvictArgs a)
{
    const int units = a.c.w / 8, pair = blockIdx.y;
    const int i = (blockIdx.x * 256 + threadIdx.x) / units, u = (blockIdx.x * 256 + threadIdx.x) % units;
    if (i >= a.n_keep) return;
    const int p = a.kept[(int64_t)pair * a.n_keep + i];
    if (p < 0) return;
    const int b = pair / a.c.n_kv, h = pair - b * a.c.n_kv;
    const int src = a.tables[(int64_t)b * a.table_stride + p / a.c.page], dst = a.new_tables[(int64_t)b * a.new_stride + i / a.c.page];
    if ((unsigned)dst >= (unsigned)a.c.n_pages) return;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if ((unsigned)src < (unsigned)a.c.n_pages) {
        const int r = p & (a.c.page - 1);
        const uint8_t *row = a.c.k_row(src, h, r) + 16 * pg_unit(a.c.w, u, r);
        k = *(const uint4 *)row;
        v = *(const uint4 *)(row + a.c.v_off());
    }
    const int r = i & (a.c.page - 1);
    uint8_t *row = a.c.k_row(dst, h, r) + 16 * pg_unit(a.c.w, u, r);
    *(uint4 *)row = k;
    *(uint4 *)(row + a.c.v_off()) = v;
}

}  // namespace

hipError_t launch_paged_evict(const PgEvictArgs &a, int n_seq, hipStream_t s)
{
    k_paged_choose<<<(unsigned)(n_seq * a.c.n_kv), kThreads, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t n = (int64_t)a.n_keep * (a.c.w / 8);
    k_paged_copy<<<dim3((unsigned)((n + 255) / 256), (unsigned)(n_seq * a.c.n_kv)), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
