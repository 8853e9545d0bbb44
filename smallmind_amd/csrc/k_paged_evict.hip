// k_paged_evict.hip -- eviction from the paged KV cache: of every sequence and KV head the last n_recent positions and
// those others that have received the most weight, n_keep in all, copied in their order to other pages.
//
// Mathematics.  With n positions, r = min(n_recent, n_keep, n) of them the last, m = min(n, n_keep) - r of the first n - r are chosen:
// those whose weight is above the m-th largest, and of those equal to it the first.  The m-th largest is found digit by
// digit: weights as unsigned numbers of the same order, a count of each value of the leading 11 bits, of the next 11 among
// those that lead alike, and of the last 10; it ends early where a digit's count is the number still wanted, for weights that differ
// mostly after two.  A NaN counts as less than every number, -0 as 0.
//
// Layout.  Choosing: one workgroup per (sequence, KV head), 64 positions at a time a wave, so that loads and stores are of
// whole lines and ballots give every position its place in order.  Up to 16384 positions the weights stay in registers;
// longer sequences are gone through a segment at a time and read again for each digit (from the L2).  What bounds it is the workgroup's own
// chain of loads, counts and barriers: 8.9 us for 700 positions, 18.6 us for 128 sequences and heads of 8192 (20 to 27 us when the
// number was found bit by bit with ballots, 21 us with 8-bit digits and positions in order of the threads).
// Copying: a lane per 16-byte unit, rows anywhere in the pages.  By the workgroup that chose where that is at most 128 KB of new
// rows, so that a second launch is spared (64 KB: 11.2 us for 8.9 + 3.4); by a launch of its own above (1 MB: 118 us for
// 18.6 + 52, of which 52 are 134 MB read and as much written at 5.2 TB/s, a large copy's rate).
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

// Lanes before this one whose bit is set.
__device__ __forceinline__ uint32_t before(uint64_t m)
{
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0u));
}

// What a workgroup works on, and what it keeps of it.
struct Job {
    int b, h, n, keep, recent, cand;
    uint32_t want;      // of the first `cand` positions
    const float *mass;
    int32_t *kept;
    float *out;

    __device__ __forceinline__ explicit Job(const PgEvictArgs &a)
    {
        b = blockIdx.x / a.c.n_kv, h = blockIdx.x - b * a.c.n_kv;
        n = min(max(a.lens[b], 0), a.max_len);
        keep = min(n, a.n_keep), recent = min(a.n_recent, keep), cand = n - recent;
        want = (uint32_t)(keep - recent);
        mass = a.mass + (int64_t)blockIdx.x * a.mass_stride;
        kept = a.kept + (int64_t)blockIdx.x * a.n_keep;
        out = a.new_mass + (int64_t)blockIdx.x * a.n_keep;
        if (h == 0 && threadIdx.x == 0) a.new_lens[b] = keep;
    }
    // The last positions, and the places that stay empty.
    __device__ __forceinline__ void rest(int n_keep) const
    {
        for (int i = threadIdx.x; i < recent; i += kThreads) {
            kept[want + i] = cand + i;
            out[want + i] = mass[cand + i];
        }
        for (int i = keep + threadIdx.x; i < n_keep; i += kThreads) {
            kept[i] = -1;
            out[i] = 0.0f;
        }
    }
};

// A wave's keys: key i of a lane is that of position first + 64 i + lane, for i < per, so that loads and stores are of whole lines
// and a ballot has 64 positions in their order.  A place without a candidate has a NaN's key.
struct Keys {
    uint32_t key[kSeg];
    int first, per, cand;

    __device__ __forceinline__ void load(const float *mass, int first_, int per_, int cand_)
    {
        first = first_, per = per_, cand = cand_;
#pragma unroll
        for (int i = 0; i < kSeg; i++) {
            const int p = first + 64 * i + (threadIdx.x & 63);
            key[i] = i < per && p < cand ? order_of(mass[p]) : 0u;
        }
    }
    __device__ __forceinline__ bool in(int i) const { return first + 64 * i + (int)(threadIdx.x & 63) < cand; }
};

// In order of position, every key above `least` and the first `ties` equal to it go to their places.  eq, at: keys equal to `least`
// and places taken in the segments before.
struct Counts {
    uint32_t gt[16], eq[16];
};
__device__ __forceinline__ void place(Counts &S, const Keys &k, const Job &j, uint32_t least, uint32_t ties, bool all, uint32_t &eq_all, uint32_t &at_all)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t gt = 0, eq = 0;
#pragma unroll
    for (int i = 0; i < kSeg; i++) {
        if (i < k.per) {
            gt += (uint32_t)__popcll(__ballot(k.in(i) && (all || k.key[i] > least)));
            eq += (uint32_t)__popcll(__ballot(k.in(i) && !all && k.key[i] == least));
        }
    }
    if (lane == 0) S.gt[wave] = gt, S.eq[wave] = eq;
    __syncthreads();
    uint32_t gb = 0, eb = 0, gall = 0, eall = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        if (w == wave) gb = gall, eb = eall;
        gall += S.gt[w], eall += S.eq[w];
    }
    eb += eq_all;
    uint32_t at = at_all + gb + min(eb, ties) - min(eq_all, ties);   // (of this wave's first)
#pragma unroll
    for (int i = 0; i < kSeg; i++) {
        if (i < k.per) {
            const bool is_eq = k.in(i) && !all && k.key[i] == least;
            const uint64_t eqs = __ballot(is_eq);
            const bool keep = (k.in(i) && (all || k.key[i] > least)) || (is_eq && eb + before(eqs) < ties);
            const uint64_t keeps = __ballot(keep);
            if (keep) {
                const int p = k.first + 64 * i + lane;
                const uint32_t to = at + before(keeps);
                j.kept[to] = p;
                j.out[to] = j.mass[p];
            }
            at += (uint32_t)__popcll(keeps);
            eb += (uint32_t)__popcll(eqs);
        }
    }
    at_all += gall + min(eq_all + eall, ties) - min(eq_all, ties);
    eq_all += eall;
    __syncthreads();
}

// Unit u of row p of the old pages to row i of the new ones.
__device__ __forceinline__ void copy_unit(const PgEvictArgs &a, int b, int h, int p, int i, int u)
{
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

// COPY: the rows too.
template <bool COPY>
__global__ __launch_bounds__(kThreads) void k_paged_choose(const PgEvictArgs a)
{
    __shared__ uint32_t hist[2048], sums[16], found[3];
    __shared__ Counts S;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Job j(a);
    const bool one = j.cand <= kSegment;                     // the keys stay in registers
    const int per = one ? (j.cand + kThreads - 1) / kThreads : kSeg, step = per * kThreads;
    Keys k;
    k.load(j.mass, wave * 64 * per, per, j.cand);
    const bool all = j.want >= (uint32_t)j.cand;
    uint32_t least = 0, ties = 0;       // the m-th largest, and how many equal to it are kept
    if (j.want > 0 && !all) {
        uint32_t left = j.want;
        hist[tid] = 0, hist[tid + kThreads] = 0;
        __syncthreads();
#pragma unroll
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, above_shift = pass == 1 ? 21 : 10;
            const uint32_t mask = pass == 2 ? 1023u : 2047u;
            for (int s0 = 0; s0 < j.cand; s0 += step) {
                if (!one) k.load(j.mass, s0 + wave * 64 * per, per, j.cand);
#pragma unroll
                for (int i = 0; i < kSeg; i++) {
                    if (i < per && k.in(i) && (pass == 0 || ((k.key[i] ^ least) >> above_shift) == 0)) {
                        const uint32_t digit = (k.key[i] >> shift) & mask;
                        // (equal weights are common, and would wait for each other)
                        const uint32_t lead = __builtin_amdgcn_readfirstlane(digit);
                        if (digit == lead) {
                            const uint64_t same = __ballot(true);
                            if (before(same) == 0) atomicAdd(&hist[digit], (uint32_t)__popcll(same));
                        } else {
                            atomicAdd(&hist[digit], 1u);
                        }
                    }
                }
            }
            __syncthreads();
            // the largest digit with `left` or more at or above it: digits from the highest down, two of a thread
            const int d0 = 2047 - 2 * tid;
            const uint32_t c0 = hist[d0], c1 = hist[d0 - 1];
            hist[d0] = 0, hist[d0 - 1] = 0;
            uint32_t sum = c0 + c1;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t v = __shfl_up(sum, o, 64);
                if (lane >= o) sum += v;
            }
            if (lane == 63) sums[wave] = sum;
            __syncthreads();
            uint32_t above = sum - c0 - c1;
#pragma unroll
            for (int w = 0; w < 16; w++) above += w < wave ? sums[w] : 0u;
            if (above < left && above + c0 >= left) found[0] = d0, found[1] = above, found[2] = c0;
            above += c0;
            if (above < left && above + c1 >= left) found[0] = d0 - 1, found[1] = above, found[2] = c1;
            __syncthreads();
            least |= found[0] << shift;
            left -= found[1];
            ties = left;
            if (found[2] == left) {     // all with these digits are kept
                ties = ~0u;
                break;
            }
        }
    }
    uint32_t eq = 0, at = 0;
    for (int s0 = 0; s0 < j.cand && j.want > 0; s0 += step) {
        if (!one) k.load(j.mass, s0 + wave * 64 * per, per, j.cand);
        place(S, k, j, least, ties, all, eq, at);
    }
    j.rest(a.n_keep);
    if constexpr (COPY) {
        __syncthreads();   // (what the workgroup has written, it reads)
        const int units = a.c.w / 8;
        for (int i = tid; i < j.keep * units; i += kThreads) copy_unit(a, j.b, j.h, j.kept[i / units], i / units, i % units);
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
    const int b = pair / a.c.n_kv;
    copy_unit(a, b, pair - b * a.c.n_kv, p, i, u);
}

}  // namespace

hipError_t launch_paged_evict(const PgEvictArgs &a, int n_seq, hipStream_t s)
{
    const unsigned pairs = (unsigned)(n_seq * a.c.n_kv);
    const bool copy = (int64_t)a.n_keep * a.c.w * 4 <= (128 << 10);   // K and V rows, 2 bytes a dim
    if (copy) k_paged_choose<true><<<pairs, kThreads, 0, s>>>(a);
    else k_paged_choose<false><<<pairs, kThreads, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || copy) return e;
    const int64_t n = (int64_t)a.n_keep * (a.c.w / 8);
    k_paged_copy<<<dim3((unsigned)((n + 255) / 256), pairs), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
