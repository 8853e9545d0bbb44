// paged_ops.cpp -- C-ABI of the paged KV cache, the attention over it, received weights and eviction.  Every argument
// that the host can see is checked here; places, page tables, positions, lengths and starts lie in device memory and are
// checked by the kernels, which never leave the cache or a row.
#include <math.h>
#include <stdio.h>

#include <new>

#include "smx_internal.h"

using namespace smx;

#define SMX_FAIL(code, ...)                                          \
    do {                                                             \
        char _b[512];                                                \
        snprintf(_b, sizeof(_b), __VA_ARGS__);                       \
        set_error(_b);                                               \
        return (code);                                               \
    } while (0)

#define SMX_HIP(expr)                                                                       \
    do {                                                                                    \
        hipError_t _e = (expr);                                                             \
        if (_e != hipSuccess) SMX_FAIL(_e == hipErrorOutOfMemory ? SMX_ENOMEM : SMX_EDEVICE, \
                                       "%s: %s", #expr, hipGetErrorString(_e));             \
    } while (0)

struct smx_paged_cache {
    int device = 0;
    PgView view{};
};

namespace {

constexpr int64_t kMaxOutputs = INT64_C(0x7FFFFFFF);
constexpr int64_t kMaxBlocks = (1 << 23) - 1;   // of up to 512 threads: a launch has fewer than 2^32
constexpr int kMaxLen = 1 << 24;

int elem_type(int type) { return type == SMX_TYPE_F32 ? PG_F32 : type == SMX_TYPE_F16 ? PG_F16 : type == SMX_TYPE_BF16 ? PG_BF16 : -1; }
int elem_bytes(int pg) { return pg == PG_F32 ? 4 : 2; }
int cache_type(const PgView &v) { return v.bf16 ? PG_BF16 : PG_F16; }
bool misaligned(const void *p, int bytes) { return (uintptr_t)p % bytes != 0; }

// Whether `bytes` bytes from p on meet one of the n rows of `row` elements of `size` bytes, `stride` elements apart, from q on.  (All are
// positive, and stride no less than row; of one row it may be anything.)
bool meet(const void *p, int64_t bytes, const void *q, int64_t n, int64_t stride, int64_t row, int size)
{
    const __int128 step = (__int128)stride * size, at = (__int128)(uintptr_t)p - (uintptr_t)q, far = at - row * size;
    const __int128 i = far < 0 ? 0 : far / step + 1;   // the first row that ends behind p
    return i < n && i * step < at + bytes;
}

// The cache's memory is on its device, so the call's stream has to be too.
int check_device(const smx_paged_cache *c, const char *fn)
{
    int dev = -1;
    SMX_HIP(hipGetDevice(&dev));
    if (dev != c->device) SMX_FAIL(SMX_EINVAL, "%s: the cache is on device %d, the current device is %d", fn, c->device, dev);
    return SMX_OK;
}

int check_rotation(const smx_rotation *r, const int32_t *pos, int head_dim, const char *fn, PgRotation *out)
{
    *out = PgRotation{};
    if (!r) return SMX_OK;
    if (!r->cos_dev || !r->sin_dev || !pos) SMX_FAIL(SMX_EINVAL, "%s: the rotation needs tables and positions", fn);
    if (misaligned(r->cos_dev, 4) || misaligned(r->sin_dev, 4) || misaligned(pos, 4)) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (r->n_pos <= 0) SMX_FAIL(SMX_EINVAL, "%s: n_pos %d must be positive", fn, r->n_pos);
    if (r->n_rot <= 0 || r->n_rot % 2 || r->n_rot > head_dim)
        SMX_FAIL(SMX_EINVAL, "%s: n_rot %d must be even and at most head_dim %d", fn, r->n_rot, head_dim);
    if (r->halves != 0 && r->halves != 1) SMX_FAIL(SMX_EINVAL, "%s: halves must be 0 or 1", fn);
    if (r->n_axes < 1 || r->n_axes > 4) SMX_FAIL(SMX_EINVAL, "%s: n_axes %d must be 1 to 4", fn, r->n_axes);
    const int half = r->n_rot / 2;
    int64_t sum = 0;
    for (int a = 0; a < 4; a++) {
        if (r->n_axes > 1 && a < r->n_axes) {
            if (r->sections[a] < 0) SMX_FAIL(SMX_EINVAL, "%s: a section is negative", fn);
            sum += r->sections[a];
        }
        out->ends[a] = a >= r->n_axes - 1 ? half : (int)(sum < half ? sum : half);
    }
    if (r->n_axes > 1 && sum != half) SMX_FAIL(SMX_EINVAL, "%s: the sections add up to %lld, not to n_rot / 2 = %d", fn, (long long)sum, half);
    out->cos = r->cos_dev;
    out->sin = r->sin_dev;
    out->pos = pos;
    out->n_pos = r->n_pos;
    out->half = half;
    out->halves = r->halves;
    out->vec = half % 4 == 0 && !misaligned(r->cos_dev, 16) && !misaligned(r->sin_dev, 16);
    return SMX_OK;
}

// Rows of queries, keys and values that a write reads; `out` is what the kernel gets.
int check_rows(int in_type, const void *q, int64_t q_stride, int n_head, const void *k, int64_t k_stride, const void *v,
               int64_t v_stride, int n_kv, int hd, const float *q_gamma, const float *k_gamma, float eps,
               const smx_rotation *rot, const int32_t *pos, int n_tok, int out_type, void *q_out, void *k_out, bool cache,
               const char *fn, PgWriteArgs *a, int *type)
{
    *a = PgWriteArgs{};
    *type = elem_type(in_type);
    a->out_type = elem_type(out_type);
    if (*type < 0 || a->out_type < 0) SMX_FAIL(SMX_EUNSUPPORTED, "%s: rows are F32, F16 or BF16", fn);
    if (hd <= 0 || hd % 8 || hd > kPgMaxHead) SMX_FAIL(SMX_EUNSUPPORTED, "%s: head_dim %d must be a multiple of 8 up to %d", fn, hd, kPgMaxHead);
    if (n_tok < 0) SMX_FAIL(SMX_EINVAL, "%s: n_tok %d is negative", fn, n_tok);
    if (q && (n_head <= 0 || n_head > 65535)) SMX_FAIL(SMX_EINVAL, "%s: n_head %d must be 1 to 65535", fn, n_head);
    if (k && (n_kv <= 0 || n_kv > 65535)) SMX_FAIL(SMX_EINVAL, "%s: n_kv_head %d must be 1 to 65535", fn, n_kv);
    if ((q && q_stride < (int64_t)n_head * hd) || (k && k_stride < (int64_t)n_kv * hd) || (v && v_stride < (int64_t)n_kv * hd))
        SMX_FAIL(SMX_EINVAL, "%s: a token's rows must be at least heads * head_dim apart", fn);
    const int in = elem_bytes(*type), out = elem_bytes(a->out_type);
    if ((q && (misaligned(q, in) || misaligned(q_out, out))) || (k && misaligned(k, in)) || (v && misaligned(v, in)) ||
        (k_out && misaligned(k_out, out)) || misaligned(q_gamma, 4) || misaligned(k_gamma, 4))
        SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (((q && q_gamma) || (k && k_gamma)) && !(eps >= 0.0f && eps < INFINITY)) SMX_FAIL(SMX_EINVAL, "%s: eps must be finite and not negative", fn);
    if (n_tok > kMaxBlocks * 4) SMX_FAIL(SMX_EUNSUPPORTED, "%s: %d tokens are too many for one launch", fn, n_tok);
    a->q = q, a->k = k, a->v = v;
    a->q_stride = q_stride, a->k_stride = k_stride, a->v_stride = v_stride;
    a->q_gamma = q_gamma, a->k_gamma = k_gamma, a->eps = eps;
    a->q_out = q_out, a->k_out = k_out;
    a->n_tok = n_tok, a->n_head = n_head, a->n_kv = n_kv, a->hd = hd;
    // eight elements at a time: rows of head_dim, a multiple of 8, keep what their base and stride have
    const int64_t piece = 16 / in;
    a->vec = (!q || (!misaligned(q, 16) && q_stride % piece == 0 && !misaligned(q_out, 16))) &&
             (!k || (!misaligned(k, 16) && k_stride % piece == 0 && (cache || !misaligned(k_out, 16)))) &&
             (!v || (!misaligned(v, 16) && v_stride % piece == 0));
    return check_rotation(rot, pos, hd, fn, &a->rot);
}

// Outputs where inputs lie: other waves may still read there.
int check_apart(const PgWriteArgs &a, int type, const char *fn)
{
    const int in = elem_bytes(type);
    const int64_t out = elem_bytes(a.out_type), hd = a.hd;
    const auto met = [&](const void *o, int64_t heads) {
        const int64_t n = o ? a.n_tok * heads * hd * out : 0;
        return n && ((a.q && meet(o, n, a.q, a.n_tok, a.q_stride, a.n_head * hd, in)) ||
                     (a.k && meet(o, n, a.k, a.n_tok, a.k_stride, a.n_kv * hd, in)) ||
                     (a.v && meet(o, n, a.v, a.n_tok, a.v_stride, a.n_kv * hd, in)));
    };
    if (met(a.q ? a.q_out : nullptr, a.n_head) || met(a.k ? a.k_out : nullptr, a.n_kv)) SMX_FAIL(SMX_EINVAL, "%s: an output lies in the inputs' memory", fn);
    return SMX_OK;
}

// What an attention call and one for received weights have in common; `a` gets it.
int check_batch(const smx_paged_cache *c, int type, int n_tok, int n_head, int n_seq, int max_q, int max_len, const char *fn)
{
    const PgView &v = c->view;
    const int t = elem_type(type);
    if (t != PG_F32 && t != cache_type(v)) SMX_FAIL(SMX_EUNSUPPORTED, "%s: q is F32 or of the cache's type", fn);
    if (n_head <= 0 || n_head % v.n_kv) SMX_FAIL(SMX_EINVAL, "%s: n_head %d must be a multiple of the cache's %d KV heads", fn, n_head, v.n_kv);
    if (n_head > 65535) SMX_FAIL(SMX_EUNSUPPORTED, "%s: more than 65535 heads", fn);
    if (n_tok < 0 || n_seq <= 0 || max_q <= 0) SMX_FAIL(SMX_EINVAL, "%s: need n_tok >= 0, n_seq >= 1 and max_q >= 1", fn);
    if (max_len < 0) SMX_FAIL(SMX_EINVAL, "%s: max_len %d is negative", fn, max_len);
    if (max_len > kMaxLen) SMX_FAIL(SMX_EUNSUPPORTED, "%s: more than 2^24 positions", fn);
    if ((double)n_tok * n_head * v.hd > (double)kMaxOutputs) SMX_FAIL(SMX_EUNSUPPORTED, "%s: %d tokens of %d heads are too many outputs", fn, n_tok, n_head);
    if ((int64_t)n_seq * v.n_kv > kMaxBlocks) SMX_FAIL(SMX_EUNSUPPORTED, "%s: too many sequences for one launch", fn);
    return SMX_OK;
}

// The factors of the scores: products to exponents of 2, or to what tanh takes and from there.
double scale_of(const PgView &v, const smx_attention_rules *r) { return r && r->scale > 0.0f ? (double)r->scale : 1.0 / sqrt((double)v.hd); }
constexpr double kLog2e = 1.4426950408889634;

int check_rules(const smx_paged_cache *c, const smx_attention_rules *r, const char *fn)
{
    if (!r) return SMX_OK;
    if (!(r->scale >= 0.0f && r->scale < INFINITY) || !(r->cap >= 0.0f && r->cap < INFINITY))
        SMX_FAIL(SMX_EINVAL, "%s: scale and cap must be finite and not negative", fn);
    const double scale = scale_of(c->view, r);
    if (scale * kLog2e > 1e37 || r->cap * kLog2e > 1e37 || (r->cap > 0.0f && scale / r->cap > 1e37))
        SMX_FAIL(SMX_EUNSUPPORTED, "%s: scale, cap or scale / cap is above the range of fp32", fn);
    if (r->window < 0) SMX_FAIL(SMX_EINVAL, "%s: window %d is negative", fn, r->window);
    if (r->reserved != 0) SMX_FAIL(SMX_EINVAL, "%s: reserved must be zero", fn);
    if (misaligned(r->slopes_dev, 4) || misaligned(r->prefix_dev, 4)) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    return SMX_OK;
}

// (a window of max_len and more hides nothing)
int window_of(const smx_attention_rules *r, int max_len) { return r && r->window < max_len ? r->window : 0; }

AttnPgArgs batch_args(const smx_paged_cache *c, int type, const void *q, int64_t q_stride, int n_tok, int n_head, int n_seq,
                      const int32_t *starts, const int32_t *lens, const int32_t *tables, int table_stride, int max_q, int max_len,
                      const smx_attention_rules *r)
{
    AttnPgArgs a{};
    const PgView &v = c->view;
    a.c = v;
    a.q = q;
    a.q_stride = q_stride;
    a.starts = starts, a.lens = lens, a.tables = tables;
    a.table_stride = table_stride;
    a.page_shift = __builtin_ctz((unsigned)v.page);
    a.n_tok = n_tok, a.n_head = n_head, a.n_seq = n_seq;
    a.group = n_head / v.n_kv;
    a.inv_group = (double)v.n_kv / n_head;
    a.max_q = max_q < n_tok ? max_q : n_tok, a.max_len = max_len;
    a.io = elem_type(type);
    const double scale = scale_of(v, r);
    a.scale_log2e = (float)(scale * kLog2e);
    // (the unit is some 2^-14 of the largest of a row: with a factor of 0 what is masked, -inf, would be NaN; scores of rows below this are
    // below 2^-70, as good as 0)
    a.q_least = (float)fmax(ldexp(1.0, -100), ldexp(1.0, -112) / (scale * kLog2e));
    if (r) {
        // (a cap so large that scale / cap leaves fp32's normal numbers changes no score of products below 2^113 by 2^-24 of itself)
        if (r->cap > 0.0f && scale / r->cap >= 1.17549435e-38) a.cap_in = (float)(scale / r->cap), a.cap_out = (float)(r->cap * kLog2e);
        a.slopes = r->slopes_dev;
        a.prefix = r->prefix_dev;
        a.window = window_of(r, max_len);
    }
    const int piece = a.io == PG_F32 ? 4 : 8;
    a.q_vec = !misaligned(q, 16) && q_stride % piece == 0;
    return a;
}

int check_operands(const smx_paged_cache *c, int type, const void *q, int64_t q_stride, int n_head, const int32_t *starts,
                   const int32_t *lens, const int32_t *tables, int table_stride, int max_len, const char *fn)
{
    if (q_stride < (int64_t)n_head * c->view.hd) SMX_FAIL(SMX_EINVAL, "%s: q_stride %lld is less than n_head * head_dim", fn, (long long)q_stride);
    if (misaligned(q, elem_bytes(elem_type(type))) || misaligned(starts, 4) || misaligned(lens, 4) || misaligned(tables, 4))
        SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (table_stride < 0 || (int64_t)table_stride * c->view.page < max_len)
        SMX_FAIL(SMX_EINVAL, "%s: %d pages of %d positions in a table are fewer than max_len %d", fn, table_stride, c->view.page, max_len);
    return SMX_OK;
}

int check_work(const void *work, int64_t have, int64_t need, const char *fn)
{
    if ((uintptr_t)work & 15) SMX_FAIL(SMX_EINVAL, "%s: the work memory must be 16-byte aligned", fn);
    if (need > 0 && (!work || have < need))
        SMX_FAIL(SMX_EINVAL, "%s: needs %lld bytes of work memory, has %lld", fn, (long long)need, (long long)(work ? have : 0));
    return SMX_OK;
}

// The plan of an attention call that has tokens and positions.
int plan_attention(const smx_paged_cache *c, int type, int n_tok, int n_head, int n_seq, int max_q, int max_len,
                   const smx_attention_rules *r, const char *fn, AttnPgPlan *p)
{
    *p = attn_paged_plan(c->view, elem_type(type), n_tok, n_head, n_seq, max_q < n_tok ? max_q : n_tok, max_len,
                         window_of(r, max_len));
    if (p->blocks > kMaxBlocks) SMX_FAIL(SMX_EUNSUPPORTED, "%s: too many workgroups for one launch", fn);
    return SMX_OK;
}

int plan_mass(const smx_paged_cache *c, int type, int n_head, int n_seq, int max_q, int max_len, const char *fn, MassPgPlan *p)
{
    const bool fits = (double)n_seq * c->view.n_kv * max_len <= (double)kMaxOutputs;   // (the plan's numbers then do as well)
    if (fits) *p = attn_mass_plan(c->view, elem_type(type), n_head, n_seq, max_q, max_len);
    if (!fits || p->blocks > kMaxBlocks)
        SMX_FAIL(SMX_EUNSUPPORTED, "%s: %d sequences of %d positions are too many outputs", fn, n_seq, max_len);
    return SMX_OK;
}

}  // namespace

extern "C" {

SMX_API int smx_paged_cache_create(int type, int n_pages, int n_kv_head, int head_dim, int page_size, smx_paged_cache **out)
{
    if (!out) SMX_FAIL(SMX_EINVAL, "smx_paged_cache_create: null out");
    *out = nullptr;
    if (type != SMX_TYPE_F16 && type != SMX_TYPE_BF16) SMX_FAIL(SMX_EUNSUPPORTED, "smx_paged_cache_create: a cache is F16 or BF16");
    if (n_pages <= 0 || n_kv_head <= 0) SMX_FAIL(SMX_EINVAL, "smx_paged_cache_create: sizes must be positive");
    if (head_dim <= 0 || head_dim % 8 || head_dim > kPgMaxHead)
        SMX_FAIL(SMX_EUNSUPPORTED, "smx_paged_cache_create: head_dim %d must be a multiple of 8 up to %d", head_dim, kPgMaxHead);
    if (page_size < kPgGroup || page_size > 1024 || (page_size & (page_size - 1)))
        SMX_FAIL(SMX_EUNSUPPORTED, "smx_paged_cache_create: page_size %d must be a power of two from 16 to 1024", page_size);
    if ((int64_t)n_pages * page_size > 0x7FFFFFFF || n_kv_head > 65535)
        SMX_FAIL(SMX_EUNSUPPORTED, "smx_paged_cache_create: more than 2^31 - 1 positions, or 65535 KV heads");
    PgView v{};
    v.n_pages = n_pages;
    v.n_kv = n_kv_head;
    v.hd = head_dim;
    v.w = pg_width(head_dim);
    v.page = page_size;
    v.bf16 = type == SMX_TYPE_BF16;
    if ((double)n_pages * n_kv_head * (double)v.head_bytes() > 1e15)
        SMX_FAIL(SMX_ENOMEM, "smx_paged_cache_create: the cache would take more than 10^15 bytes");
    smx_paged_cache *c = new (std::nothrow) smx_paged_cache();
    if (!c) SMX_FAIL(SMX_ENOMEM, "smx_paged_cache_create: out of host memory");
    c->view = v;
    hipError_t e = hipGetDevice(&c->device);
    if (e == hipSuccess) e = hipMalloc((void **)&c->view.base, v.bytes());
    // zeros: what was never written, and what lies beyond head_dim, weighs nothing and is finite
    if (e == hipSuccess) e = hipMemset(c->view.base, 0, v.bytes());
    if (e == hipSuccess) e = hipDeviceSynchronize();
    if (e != hipSuccess) {
        if (c->view.base) (void)hipFree(c->view.base);
        delete c;
        (void)hipGetLastError();   // reported here; the check after the next launch is not to find it again
        SMX_HIP(e);
    }
    *out = c;
    return SMX_OK;
}

SMX_API int smx_paged_cache_info(const smx_paged_cache *c, int *type, int *n_pages, int *n_kv_head, int *head_dim, int *page_size,
                                 int64_t *bytes)
{
    if (!c) SMX_FAIL(SMX_EINVAL, "smx_paged_cache_info: null cache");
    if (type) *type = c->view.bf16 ? SMX_TYPE_BF16 : SMX_TYPE_F16;
    if (n_pages) *n_pages = c->view.n_pages;
    if (n_kv_head) *n_kv_head = c->view.n_kv;
    if (head_dim) *head_dim = c->view.hd;
    if (page_size) *page_size = c->view.page;
    if (bytes) *bytes = (int64_t)c->view.bytes();
    return SMX_OK;
}

SMX_API int smx_paged_cache_destroy(smx_paged_cache *c)
{
    if (!c) return SMX_OK;
    int dev = -1;
    const bool moved = hipGetDevice(&dev) == hipSuccess && dev != c->device && hipSetDevice(c->device) == hipSuccess;
    const hipError_t e = hipFree(c->view.base);   // waits for the device's queued work
    if (moved) (void)hipSetDevice(dev);
    delete c;
    SMX_HIP(e);
    return SMX_OK;
}

SMX_API int smx_qk_norm_rope(int in_type, const void *q_dev, int64_t q_stride, int n_head, const void *k_dev, int64_t k_stride,
                             int n_kv_head, int head_dim, const float *q_gamma_dev, const float *k_gamma_dev, float eps,
                             const smx_rotation *rot, const int32_t *pos_dev, int n_tok, int out_type, void *q_out_dev,
                             void *k_out_dev, void *stream)
{
    const char *fn = "smx_qk_norm_rope";
    if ((!q_dev && !k_dev) || (q_dev && !q_out_dev) || (k_dev && !k_out_dev)) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    PgWriteArgs a;
    int type;
    int rc = check_rows(in_type, q_dev, q_stride, n_head, k_dev, k_stride, nullptr, 0, n_kv_head, head_dim, q_gamma_dev,
                              k_gamma_dev, eps, rot, pos_dev, n_tok, out_type, q_out_dev, k_out_dev, false, fn, &a, &type);
    if (rc != SMX_OK || n_tok == 0 || (rc = check_apart(a, type, fn)) != SMX_OK) return rc;
    SMX_HIP(launch_paged_write(a, type, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_paged_append(smx_paged_cache *c, int in_type, const void *q_dev, int64_t q_stride, int n_head, const void *k_dev,
                             int64_t k_stride, const void *v_dev, int64_t v_stride, const float *q_gamma_dev,
                             const float *k_gamma_dev, float eps, const smx_rotation *rot, const int32_t *pos_dev,
                             const int32_t *places_dev, int n_tok, int out_type, void *q_out_dev, void *stream)
{
    const char *fn = "smx_paged_append";
    if (!c || !k_dev || !v_dev || !places_dev || (q_dev && !q_out_dev)) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    PgWriteArgs a;
    int type, rc = check_rows(in_type, q_dev, q_stride, n_head, k_dev, k_stride, v_dev, v_stride, c->view.n_kv, c->view.hd,
                              q_gamma_dev, k_gamma_dev, eps, rot, pos_dev, n_tok, out_type, q_out_dev, nullptr, true, fn, &a, &type);
    if (rc != SMX_OK) return rc;
    if (misaligned(places_dev, 4)) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (n_tok == 0) return SMX_OK;
    if ((rc = check_apart(a, type, fn)) != SMX_OK || (rc = check_device(c, fn)) != SMX_OK) return rc;
    a.c = c->view;
    a.places = places_dev;
    SMX_HIP(launch_paged_write(a, type, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_paged_read(const smx_paged_cache *c, const int32_t *places_dev, int n_tok, void *k_dev, void *v_dev, void *stream)
{
    const char *fn = "smx_paged_read";
    if (!c || !places_dev || !k_dev || !v_dev) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    if (misaligned(k_dev, 16) || misaligned(v_dev, 16) || misaligned(places_dev, 4)) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (n_tok < 0) SMX_FAIL(SMX_EINVAL, "%s: n_tok %d is negative", fn, n_tok);
    if ((int64_t)n_tok * c->view.n_kv > kMaxBlocks * 8) SMX_FAIL(SMX_EUNSUPPORTED, "%s: %d tokens are too many for one launch", fn, n_tok);
    if (n_tok == 0) return SMX_OK;
    const int rc = check_device(c, fn);
    if (rc != SMX_OK) return rc;
    SMX_HIP(launch_paged_read(c->view, places_dev, n_tok, k_dev, v_dev, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_attention_paged_work_bytes(const smx_paged_cache *c, int type, int n_tok, int n_head, int n_seq, int max_q,
                                           int max_len, const smx_attention_rules *rules, int64_t *bytes)
{
    const char *fn = "smx_attention_paged_work_bytes";
    if (!c || !bytes) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    int rc = check_batch(c, type, n_tok, n_head, n_seq, max_q, max_len, fn);
    if (rc != SMX_OK || (rc = check_rules(c, rules, fn)) != SMX_OK) return rc;
    *bytes = 0;
    if (n_tok == 0) return SMX_OK;
    AttnPgPlan p;
    rc = plan_attention(c, type, n_tok, n_head, n_seq, max_q, max_len, rules, fn, &p);
    if (rc == SMX_OK) *bytes = p.work_bytes;
    return rc;
}

SMX_API int smx_attention_mass_work_bytes(const smx_paged_cache *c, int type, int n_head, int n_seq, int max_q, int max_len, int64_t *bytes)
{
    const char *fn = "smx_attention_mass_work_bytes";
    if (!c || !bytes) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    int rc = check_batch(c, type, 0, n_head, n_seq, max_q, max_len, fn);
    if (rc != SMX_OK) return rc;
    *bytes = 0;
    if (max_len == 0) return SMX_OK;
    MassPgPlan p;
    rc = plan_mass(c, type, n_head, n_seq, max_q, max_len, fn, &p);
    if (rc == SMX_OK) *bytes = p.work_bytes;
    return rc;
}

SMX_API int smx_attention_paged(const smx_paged_cache *c, int type, const void *q_dev, int64_t q_stride, void *out_dev,
                                float *lse_dev, int n_tok, int n_head, int n_seq, const int32_t *starts_dev,
                                const int32_t *lens_dev, const int32_t *tables_dev, int table_stride, int max_q, int max_len,
                                const smx_attention_rules *rules, void *work_dev, int64_t work_bytes, void *stream)
{
    const char *fn = "smx_attention_paged";
    if (!c || (n_tok > 0 && (!q_dev || !out_dev)) || !starts_dev || !lens_dev || (max_len > 0 && !tables_dev)) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    int rc = check_batch(c, type, n_tok, n_head, n_seq, max_q, max_len, fn);
    if (rc != SMX_OK || (rc = check_rules(c, rules, fn)) != SMX_OK) return rc;
    if ((rc = check_operands(c, type, q_dev, q_stride, n_head, starts_dev, lens_dev, tables_dev, table_stride, max_len, fn)) != SMX_OK) return rc;
    if (misaligned(out_dev, elem_bytes(elem_type(type))) || misaligned(lse_dev, 4)) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (n_tok == 0) return SMX_OK;
    AttnPgPlan p;
    if ((rc = plan_attention(c, type, n_tok, n_head, n_seq, max_q, max_len, rules, fn, &p)) != SMX_OK) return rc;
    if ((rc = check_work(work_dev, work_bytes, p.work_bytes, fn)) != SMX_OK) return rc;
    const int size = elem_bytes(elem_type(type));
    const int64_t rows = (int64_t)n_tok * n_head, hd = c->view.hd;
    if (meet(out_dev, rows * hd * size, q_dev, n_tok, q_stride, n_head * hd, size) ||
        (lse_dev && meet(lse_dev, rows * 4, q_dev, n_tok, q_stride, n_head * hd, size)))
        SMX_FAIL(SMX_EINVAL, "%s: an output lies in q's memory", fn);
    if ((rc = check_device(c, fn)) != SMX_OK) return rc;
    AttnPgArgs a = batch_args(c, type, q_dev, q_stride, n_tok, n_head, n_seq, starts_dev, lens_dev, tables_dev, table_stride, max_q,
                              max_len, rules);
    a.out = out_dev;
    a.lse = lse_dev;
    a.out_vec = !misaligned(out_dev, 16);
    SMX_HIP(launch_attn_paged(a, p, p.work_bytes > 0 ? work_dev : nullptr, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_attention_mass(const smx_paged_cache *c, int type, const void *q_dev, int64_t q_stride, const float *lse_dev,
                               const float *mass_dev, int64_t mass_stride, int mass_width, float *mass_out_dev, int n_tok,
                               int n_head, int n_seq, const int32_t *starts_dev, const int32_t *lens_dev,
                               const int32_t *tables_dev, int table_stride, int max_q, int max_len,
                               const smx_attention_rules *rules, void *work_dev, int64_t work_bytes, void *stream)
{
    const char *fn = "smx_attention_mass";
    if (!c || (n_tok > 0 && (!q_dev || !lse_dev)) || !mass_out_dev || !starts_dev || !lens_dev || (max_len > 0 && !tables_dev)) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    int rc = check_batch(c, type, n_tok, n_head, n_seq, max_q, max_len, fn);
    if (rc != SMX_OK || (rc = check_rules(c, rules, fn)) != SMX_OK) return rc;
    if ((rc = check_operands(c, type, q_dev, q_stride, n_head, starts_dev, lens_dev, tables_dev, table_stride, max_len, fn)) != SMX_OK) return rc;
    if (mass_dev && (mass_width < 0 || mass_stride < mass_width)) SMX_FAIL(SMX_EINVAL, "%s: rows of mass must be at least mass_width apart", fn);
    if (mass_dev == mass_out_dev && mass_stride != max_len) SMX_FAIL(SMX_EINVAL, "%s: in place, rows of mass must be max_len apart", fn);
    if (misaligned(lse_dev, 4) || misaligned(mass_dev, 4) || misaligned(mass_out_dev, 4)) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if (max_len == 0) return SMX_OK;
    const int64_t pairs = (int64_t)n_seq * c->view.n_kv;
    if (mass_dev && mass_dev != mass_out_dev && mass_width > 0 && meet(mass_out_dev, pairs * max_len * 4, mass_dev, pairs, mass_stride, mass_width, 4))
        SMX_FAIL(SMX_EINVAL, "%s: mass and mass_out overlap", fn);
    MassPgPlan p;
    if ((rc = plan_mass(c, type, n_head, n_seq, max_q, max_len, fn, &p)) != SMX_OK) return rc;
    if ((rc = check_work(work_dev, work_bytes, p.work_bytes, fn)) != SMX_OK) return rc;
    if ((rc = check_device(c, fn)) != SMX_OK) return rc;
    AttnPgArgs a = batch_args(c, type, q_dev, q_stride, n_tok, n_head, n_seq, starts_dev, lens_dev, tables_dev, table_stride, max_q,
                              max_len, rules);
    a.lse_in = lse_dev;
    a.mass = mass_dev;
    a.mass_stride = mass_stride;
    a.mass_width = mass_width;
    a.mass_out = mass_out_dev;
    SMX_HIP(launch_attn_mass(a, p, p.work_bytes > 0 ? work_dev : nullptr, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_paged_evict(smx_paged_cache *c, const float *mass_dev, int64_t mass_stride, const int32_t *lens_dev, int n_seq,
                            int max_len, int n_keep, int n_recent, const int32_t *tables_dev, int table_stride,
                            const int32_t *new_tables_dev, int new_stride, int32_t *kept_dev, int32_t *new_lens_dev,
                            float *new_mass_dev, void *stream)
{
    const char *fn = "smx_paged_evict";
    if (!c || !mass_dev || !lens_dev || !tables_dev || !new_tables_dev || !kept_dev || !new_lens_dev || !new_mass_dev)
        SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    if (n_seq <= 0 || max_len <= 0 || n_keep <= 0) SMX_FAIL(SMX_EINVAL, "%s: n_seq, max_len and n_keep must be positive", fn);
    if (n_recent < 0 || n_recent > n_keep) SMX_FAIL(SMX_EINVAL, "%s: n_recent %d must be 0 to n_keep %d", fn, n_recent, n_keep);
    if (max_len > kMaxLen || n_keep > kMaxLen) SMX_FAIL(SMX_EUNSUPPORTED, "%s: more than 2^24 positions", fn);
    if ((int64_t)n_seq * c->view.n_kv > 65535) SMX_FAIL(SMX_EUNSUPPORTED, "%s: more than 65535 sequences times KV heads", fn);
    if (mass_stride < max_len) SMX_FAIL(SMX_EINVAL, "%s: rows of mass must be at least max_len apart", fn);
    if (table_stride < 0 || (int64_t)table_stride * c->view.page < max_len || new_stride < 0 || (int64_t)new_stride * c->view.page < n_keep)
        SMX_FAIL(SMX_EINVAL, "%s: the tables have fewer pages than max_len or n_keep positions", fn);
    if (misaligned(mass_dev, 4) || misaligned(lens_dev, 4) || misaligned(tables_dev, 4) || misaligned(new_tables_dev, 4) ||
        misaligned(kept_dev, 4) || misaligned(new_lens_dev, 4) || misaligned(new_mass_dev, 4))
        SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    // (a head's workgroup may be done before another of the same sequence begins)
    const int64_t pairs = (int64_t)n_seq * c->view.n_kv, kept = pairs * n_keep * 4;
    const auto met = [&](const void *o, int64_t bytes) {
        return meet(o, bytes, mass_dev, pairs, mass_stride, max_len, 4) || meet(o, bytes, lens_dev, 1, n_seq, n_seq, 4) ||
               meet(o, bytes, tables_dev, 1, 1, (int64_t)n_seq * table_stride, 4) ||
               meet(o, bytes, new_tables_dev, 1, 1, (int64_t)n_seq * new_stride, 4);
    };
    if (met(kept_dev, kept) || met(new_lens_dev, (int64_t)n_seq * 4) || met(new_mass_dev, kept))
        SMX_FAIL(SMX_EINVAL, "%s: an output lies in the inputs' memory", fn);
    const int rc = check_device(c, fn);
    if (rc != SMX_OK) return rc;
    PgEvictArgs a{};
    a.c = c->view;
    a.mass = mass_dev;
    a.mass_stride = mass_stride;
    a.lens = lens_dev, a.tables = tables_dev, a.new_tables = new_tables_dev;
    a.kept = kept_dev, a.new_lens = new_lens_dev, a.new_mass = new_mass_dev;
    a.table_stride = table_stride, a.new_stride = new_stride;
    a.n_keep = n_keep, a.n_recent = n_recent, a.max_len = max_len;
    SMX_HIP(launch_paged_evict(a, n_seq, (hipStream_t)stream));
    return SMX_OK;
}

}  // extern "C"
