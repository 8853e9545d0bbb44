// k_verify.hip -- verification of drafted tokens against the target model's probabilities
// (speculative decoding).
//
// Sequence b has n drafted tokens x_0 .. x_{n-1}, the draft model's probabilities q_i they were drawn
// from, the target model's p_0 .. p_n, and uniform random numbers.  Draft i is taken if u_i q_i(x_i) <
// p_i(x_i), that is with probability min(1, p / q), up to the first that is not.  Then one token
// is drawn: from max(p_i - q_i, 0), normalised, at the draft i that was refused, or from p_n when
// none was, so that every token is distributed as the target's.  Weights and their running sums C are
// held in 64 bits and the product u_i q_i is exact there; the token is the lowest j of positive weight with
// C_j > u C_last.  Where p or q is NaN, the comparison is false and the weight 0.
//
// One workgroup of 1024 threads per sequence.  What has to be read is one row of p and one of q; a wave
// sums a stretch of the vocabulary, the wave in whose stretch the threshold falls is found from the 16
// sums, and that stretch is read again (from the cache) by all threads, a few values each.  What bounds it is
// the chain of loads that wait for one another (length, drafts' probabilities, rows, stretch) and, for
// the rows, how many a compute unit has in flight: kBatch values of each per thread.  4 drafts, 32000
// tokens: 6.3 us; 64 sequences of 7 drafts, 50257 tokens: 12 us, 26 MB.
#include "smx_device.h"
#include "smx_internal.h"

namespace smx {

namespace {

constexpr int kT = 1024;
constexpr int kW = kT / 64;
constexpr int kBatch = 16;

struct VerifyArgs {
    const float *p, *q;
    int64_t p_stride, q_stride;   // between rows
    const int32_t *draft, *lens;
    const float *u_accept, *u_draw;
    int n_draft, vocab;
    int32_t *tokens, *accepted;
};

__device__ __forceinline__ double wave_sum_f64(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

__device__ __forceinline__ double wave_scan_f64(double v, int lane)
{
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

struct VerifyShared {
    double sum[kW], scan[kW];
    int first[kW], last[kW];
};

// The token drawn with `u` from weights max(p - q, 0) (q: a row, or 1 at token `hot`, or nothing) over the
// vocabulary; -1 without a positive weight.  Called by all threads.
template <int MODE>   // 0: p alone, 1: p - q, 2: p without `hot`
__device__ __forceinline__ int draw(VerifyShared &S, const float *__restrict__ p, const float *__restrict__ q, int hot,
                                    int vocab, double u)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const auto weight = [&](int j, float pj, float qj) -> double {
        double w = (double)pj;
        if constexpr (MODE == 1) w -= (double)qj;
        if constexpr (MODE == 2) w -= j == hot ? 1.0 : 0.0;
        return fmax(w, 0.0);   // (a NaN weighs nothing)
    };
    const int seg = ((vocab + kW - 1) / kW + 63) & ~63;
    const int a = min(vocab, wave * seg), e = min(vocab, a + seg);
    double c = 0.0;
    int j0 = a + lane;
    for (; j0 - lane + 64 * kBatch <= e; j0 += 64 * kBatch) {
        const float *pj = p + j0, *qj = q + j0;
        float pv[kBatch], qv[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            pv[k] = pj[64 * k];
            if constexpr (MODE == 1) qv[k] = qj[64 * k];
        }
#pragma unroll
        for (int k = 0; k < kBatch; k++) c += weight(j0 + 64 * k, pv[k], MODE == 1 ? qv[k] : 0.0f);
    }
#pragma unroll 4
    for (; j0 < e; j0 += 64) c += weight(j0, p[j0], MODE == 1 ? q[j0] : 0.0f);
    c = wave_sum_f64(c);
    if (lane == 0) S.sum[wave] = c;
    __syncthreads();
    double total = 0.0, before = 0.0;
#pragma unroll
    for (int w = 0; w < kW; w++) total += S.sum[w];
    if (!(total > 0.0)) return -1;   // the same in every thread
    const double at = u * total;
    // the first stretch whose end passes the threshold; the last with weight where rounding hides it
    int pick = -1;
    double run = 0.0;
    bool passed = false;
#pragma unroll
    for (int w = 0; w < kW; w++) {
        const double t = S.sum[w];
        if (!passed && t > 0.0) {
            pick = w;
            before = run;
            passed = run + t > at;
        }
        run += t;
    }
    const int b0 = pick * seg, b1 = min(vocab, b0 + seg);
    // each thread a few consecutive weights of that stretch, in order
    const int per = (seg + kT - 1) / kT, f = min(b1, b0 + tid * per), l = min(b1, f + per);
    double own = 0.0;
    for (int j = f; j < l; j++) own += weight(j, p[j], MODE == 1 ? q[j] : 0.0f);
    const double upto = wave_scan_f64(own, lane);
    if (lane == 63) S.scan[wave] = upto;
    __syncthreads();
    double r = before;
#pragma unroll
    for (int w = 0; w < kW; w++) r += w < wave ? S.scan[w] : 0.0;
    r += upto - own;
    int first = -1, last = -1;
    for (int j = f; j < l; j++) {
        const double w = weight(j, p[j], MODE == 1 ? q[j] : 0.0f);
        r += w;
        if (w > 0.0) {
            last = j;
            if (first < 0 && r > at) first = j;
        }
    }
    // the lowest of all; without one (rounding hides the threshold) the last token with weight
    const uint64_t some = __ballot(first >= 0), any = __ballot(last >= 0);
    if (lane == 0) {
        S.first[wave] = some ? __builtin_amdgcn_readlane(first, __ffsll((unsigned long long)some) - 1) : vocab;
        S.last[wave] = any ? __builtin_amdgcn_readlane(last, 63 - __clzll((unsigned long long)any)) : -1;
    }
    __syncthreads();
    int lo = vocab, hi = -1;
#pragma unroll
    for (int w = 0; w < kW; w++) lo = min(lo, S.first[w]), hi = max(hi, S.last[w]);
    return lo < vocab ? lo : hi;
}

__global__ __launch_bounds__(kT) void k_verify(const VerifyArgs a)
{
    __shared__ VerifyShared S;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int n = a.lens ? min(a.lens[b], a.n_draft) : a.n_draft;
    int32_t *out = a.tokens + (int64_t)b * (a.n_draft + 1);
    const double u = (double)a.u_draw[b];
    const int32_t *x = a.draft + (int64_t)b * a.n_draft;
    const float *p = a.p + (int64_t)b * (a.n_draft + 1) * a.p_stride;
    const float *q = a.q ? a.q + (int64_t)b * a.n_draft * a.q_stride : nullptr;
    // drafts taken: every wave finds it for itself (all that can be is requested before n is known)
    int taken = max(n, 0);
    for (int i0 = 0; i0 < a.n_draft; i0 += 64) {
        const int i = i0 + lane;
        bool no = true;
        if (i < a.n_draft) {
            const int t = x[i];
            const double ua = (double)a.u_accept[(int64_t)b * a.n_draft + i];
            if ((unsigned)t < (unsigned)a.vocab) {
                const double qt = q ? (double)q[i * a.q_stride + t] : 1.0;
                no = !(ua * qt < (double)p[i * a.p_stride + t]);
            }
        }
        const uint64_t refused = __ballot(no || i >= n);
        if (refused) {
            taken = max(0, min(n, i0 + __ffsll((unsigned long long)refused) - 1));
            break;
        }
    }
    if (n < 0) {   // no sequence here
        for (int i = tid; i <= a.n_draft; i += kT) out[i] = -1;
        if (tid == 0) a.accepted[b] = 0;
        return;
    }
    const float *row = p + taken * a.p_stride;
    int tok = -1;
    if (taken < n) {
        tok = q ? draw<1>(S, row, q + taken * a.q_stride, 0, a.vocab, u) : draw<2>(S, row, nullptr, x[taken], a.vocab, u);
        __syncthreads();
    }
    // nothing left of p - q (probabilities that do not sum to 1): p itself
    if (tok < 0) tok = draw<0>(S, row, nullptr, 0, a.vocab, u);
    for (int i = tid; i <= a.n_draft; i += kT) out[i] = i < taken ? x[i] : i == taken ? tok : -1;
    if (tid == 0) a.accepted[b] = taken;
}

}  // namespace

hipError_t launch_verify(const float *p, int64_t p_stride, const float *q, int64_t q_stride, const int32_t *draft,
                         const int32_t *lens, const float *u_accept, const float *u_draw, int n_seq, int n_draft,
                         int vocab, int32_t *tokens, int32_t *accepted, hipStream_t s)
{
    const VerifyArgs a{p, q, p_stride, q_stride, draft, lens, u_accept, u_draw, n_draft, vocab, tokens, accepted};
    k_verify<<<n_seq, kT, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace smx
