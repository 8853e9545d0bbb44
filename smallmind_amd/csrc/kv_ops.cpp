// kv_ops.cpp -- C-ABI of the 8-bit KV cache, the attention over it and the verification of drafted
// tokens.  Every argument that the host can see is checked here; slots, positions, lengths and tokens
// lie in device memory and are checked by the kernels, which never leave the cache or a row.
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

struct smx_kv_cache {
    int device = 0;
    KvView view{};
};

namespace {

constexpr int64_t kMaxOutputs = INT64_C(0x7FFFFFFF);
constexpr int64_t kMaxBlocks = (1 << 24) - 1;   // of 256 threads: a launch has fewer than 2^32

// The cache's memory is on its device, so the call's stream has to be too.
int check_device(const smx_kv_cache *c, const char *fn)
{
    int dev = -1;
    SMX_HIP(hipGetDevice(&dev));
    if (dev != c->device) SMX_FAIL(SMX_EINVAL, "%s: the cache is on device %d, the current device is %d", fn, c->device, dev);
    return SMX_OK;
}

// The sizes of an attention call; `plan` says how it is cut up.
int check_attention(const smx_kv_cache *c, int n_seq, int n_q, int n_head, int prefix_len, int max_len, const char *fn,
                    AttnQ8Plan *plan)
{
    const KvView &v = c->view;
    if (n_head <= 0 || n_head % v.n_kv) SMX_FAIL(SMX_EINVAL, "%s: n_head %d must be a multiple of the cache's %d KV heads", fn, n_head, v.n_kv);
    if (n_head > 65535) SMX_FAIL(SMX_EUNSUPPORTED, "%s: more than 65535 heads", fn);
    if (n_seq <= 0 || n_q <= 0) SMX_FAIL(SMX_EINVAL, "%s: need n_seq and n_q of at least 1", fn);
    if (max_len < 0 || max_len > v.ctx || prefix_len < 0 || prefix_len > v.ctx)
        SMX_FAIL(SMX_EINVAL, "%s: max_len %d and prefix_len %d must be within 0 .. ctx %d", fn, max_len, prefix_len, v.ctx);
    if ((double)n_seq * n_q * n_head * v.hd > (double)kMaxOutputs)
        SMX_FAIL(SMX_EUNSUPPORTED, "%s: %d x %d tokens of %d heads are too many outputs", fn, n_seq, n_q, n_head);
    *plan = attn_q8_plan(v, n_seq, n_q, n_head, prefix_len, max_len);
    // (the join has fewer: at most 2^31 outputs, four per thread, and several threads for one only where rows are few)
    if (plan->blocks > kMaxBlocks) SMX_FAIL(SMX_EUNSUPPORTED, "%s: too many sequences for one launch", fn);
    return SMX_OK;
}

int attend(const smx_kv_cache *c, const float *q, int64_t q_stride, float *out, int n_seq, int n_q, int n_head,
           int prefix_slot, int prefix_len, const int32_t *slots, const int32_t *lens, int max_len, void *work,
           int64_t work_bytes, void *stream, const char *fn)
{
    if (!c || !q || !out || !slots || !lens) SMX_FAIL(SMX_EINVAL, "%s: null argument", fn);
    AttnQ8Plan plan;
    int rc = check_attention(c, n_seq, n_q, n_head, prefix_len, max_len, fn, &plan);
    if (rc != SMX_OK) return rc;
    if (prefix_len > 0 && (prefix_slot < 0 || prefix_slot >= c->view.n_slots))
        SMX_FAIL(SMX_EINVAL, "%s: prefix_slot %d of %d slots", fn, prefix_slot, c->view.n_slots);
    if (q_stride < (int64_t)n_head * c->view.hd)
        SMX_FAIL(SMX_EINVAL, "%s: q_stride %lld is less than n_head * head_dim", fn, (long long)q_stride);
    if (((uintptr_t)q | (uintptr_t)out) & 3) SMX_FAIL(SMX_EINVAL, "%s: misaligned pointer", fn);
    if ((uintptr_t)work & 15) SMX_FAIL(SMX_EINVAL, "%s: the work memory must be 16-byte aligned", fn);
    if (plan.work_bytes > 0 && (!work || work_bytes < plan.work_bytes))
        SMX_FAIL(SMX_EINVAL, "%s: needs %lld bytes of work memory, has %lld", fn, (long long)plan.work_bytes,
                 (long long)(work ? work_bytes : 0));
    if ((rc = check_device(c, fn)) != SMX_OK) return rc;
    SMX_HIP(launch_attn_q8(c->view, plan, q, q_stride, out, n_seq, n_q, n_head, prefix_slot, prefix_len, slots, lens,
                           max_len, plan.work_bytes > 0 ? work : nullptr, (hipStream_t)stream));
    return SMX_OK;
}

}  // namespace

extern "C" {

SMX_API int smx_kv_cache_create(int n_slots, int n_kv_head, int head_dim, int ctx, smx_kv_cache **out)
{
    if (!out) SMX_FAIL(SMX_EINVAL, "smx_kv_cache_create: null out");
    *out = nullptr;
    if (n_slots <= 0 || n_kv_head <= 0 || ctx <= 0) SMX_FAIL(SMX_EINVAL, "smx_kv_cache_create: sizes must be positive");
    if (head_dim <= 0 || head_dim % 8 || head_dim > kKvMaxHead)
        SMX_FAIL(SMX_EUNSUPPORTED, "smx_kv_cache_create: head_dim %d must be a multiple of 8 up to %d", head_dim, kKvMaxHead);
    if (ctx > (1 << 24) || n_kv_head > 65535 || n_slots > (1 << 24))
        SMX_FAIL(SMX_EUNSUPPORTED, "smx_kv_cache_create: more than 2^24 positions or slots, or 65535 KV heads");
    KvView v{};
    v.n_slots = n_slots;
    v.n_kv = n_kv_head;
    v.hd = head_dim;
    v.w = kv_width(head_dim);
    v.ctx = ctx;
    v.tiles = (ctx + kKvTile - 1) / kKvTile;
    if ((double)n_slots * n_kv_head * v.tiles * (double)kv_tile_bytes(v.w) > 1e15)
        SMX_FAIL(SMX_ENOMEM, "smx_kv_cache_create: the cache would take more than 10^15 bytes");
    smx_kv_cache *c = new (std::nothrow) smx_kv_cache();
    if (!c) SMX_FAIL(SMX_ENOMEM, "smx_kv_cache_create: out of host memory");
    c->view = v;
    hipError_t e = hipGetDevice(&c->device);
    if (e == hipSuccess) e = hipMalloc((void **)&c->view.base, v.bytes());
    // zero scales: a position reads as zeros until it is written
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

SMX_API int smx_kv_cache_info(const smx_kv_cache *c, int *n_slots, int *n_kv_head, int *head_dim, int *ctx, int64_t *bytes)
{
    if (!c) SMX_FAIL(SMX_EINVAL, "smx_kv_cache_info: null cache");
    if (n_slots) *n_slots = c->view.n_slots;
    if (n_kv_head) *n_kv_head = c->view.n_kv;
    if (head_dim) *head_dim = c->view.hd;
    if (ctx) *ctx = c->view.ctx;
    if (bytes) *bytes = (int64_t)c->view.bytes();
    return SMX_OK;
}

SMX_API int smx_kv_cache_destroy(smx_kv_cache *c)
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

SMX_API int smx_kv_append(smx_kv_cache *c, const float *k_dev, int64_t k_stride, const float *v_dev, int64_t v_stride,
                          const int32_t *slots_dev, const int32_t *pos_dev, int n_tok, void *stream)
{
    if (!c || !k_dev || !v_dev || !slots_dev || !pos_dev) SMX_FAIL(SMX_EINVAL, "smx_kv_append: null argument");
    const int64_t row = (int64_t)c->view.n_kv * c->view.hd;
    if (k_stride < row || v_stride < row)
        SMX_FAIL(SMX_EINVAL, "smx_kv_append: k_stride %lld and v_stride %lld must be at least n_kv_head * head_dim = %lld",
                 (long long)k_stride, (long long)v_stride, (long long)row);
    if (((uintptr_t)k_dev | (uintptr_t)v_dev) & 3) SMX_FAIL(SMX_EINVAL, "smx_kv_append: misaligned pointer");
    if (n_tok < 0 || ((int64_t)n_tok + 63) / 64 * c->view.n_kv * 2 > kMaxBlocks)
        SMX_FAIL(SMX_EINVAL, "smx_kv_append: n_tok %d out of range", n_tok);
    if (n_tok == 0) return SMX_OK;
    const int rc = check_device(c, "smx_kv_append");
    if (rc != SMX_OK) return rc;
    SMX_HIP(launch_kv_append(c->view, k_dev, k_stride, v_dev, v_stride, slots_dev, pos_dev, n_tok, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_kv_read(const smx_kv_cache *c, const int32_t *slots_dev, const int32_t *pos_dev, int n_tok, float *k_dev,
                        float *v_dev, void *stream)
{
    if (!c || !k_dev || !v_dev || !slots_dev || !pos_dev) SMX_FAIL(SMX_EINVAL, "smx_kv_read: null argument");
    if (((uintptr_t)k_dev | (uintptr_t)v_dev) & 3) SMX_FAIL(SMX_EINVAL, "smx_kv_read: misaligned pointer");
    if (n_tok < 0 || ((int64_t)n_tok + 63) / 64 * c->view.n_kv * 2 > kMaxBlocks)
        SMX_FAIL(SMX_EINVAL, "smx_kv_read: n_tok %d out of range", n_tok);
    if (n_tok == 0) return SMX_OK;
    const int rc = check_device(c, "smx_kv_read");
    if (rc != SMX_OK) return rc;
    SMX_HIP(launch_kv_read(c->view, slots_dev, pos_dev, n_tok, k_dev, v_dev, (hipStream_t)stream));
    return SMX_OK;
}

SMX_API int smx_attention_work_bytes(const smx_kv_cache *c, int n_seq, int n_q, int n_head, int prefix_len, int max_len,
                                     int64_t *bytes)
{
    if (!c || !bytes) SMX_FAIL(SMX_EINVAL, "smx_attention_work_bytes: null argument");
    AttnQ8Plan plan;
    const int rc = check_attention(c, n_seq, n_q, n_head, prefix_len, max_len, "smx_attention_work_bytes", &plan);
    if (rc == SMX_OK) *bytes = plan.work_bytes;
    return rc;
}

SMX_API int smx_attention_cached(const smx_kv_cache *c, const float *q_dev, int64_t q_stride, float *out_dev, int n_seq,
                                 int n_q, int n_head, const int32_t *slots_dev, const int32_t *lens_dev, int max_len,
                                 void *work_dev, int64_t work_bytes, void *stream)
{
    return attend(c, q_dev, q_stride, out_dev, n_seq, n_q, n_head, 0, 0, slots_dev, lens_dev, max_len, work_dev, work_bytes,
                  stream, "smx_attention_cached");
}

SMX_API int smx_attention_shared(const smx_kv_cache *c, const float *q_dev, int64_t q_stride, float *out_dev, int n_seq,
                                 int n_q, int n_head, int prefix_slot, int prefix_len, const int32_t *slots_dev,
                                 const int32_t *lens_dev, int max_len, void *work_dev, int64_t work_bytes, void *stream)
{
    return attend(c, q_dev, q_stride, out_dev, n_seq, n_q, n_head, prefix_slot, prefix_len, slots_dev, lens_dev, max_len,
                  work_dev, work_bytes, stream, "smx_attention_shared");
}

SMX_API int smx_verify_draft(const float *target_dev, int64_t target_stride, const float *draft_dev, int64_t draft_stride,
                             const int32_t *tokens_dev, const int32_t *lens_dev, const float *u_accept_dev,
                             const float *u_draw_dev, int n_seq, int n_draft, int vocab, int32_t *out_dev,
                             int32_t *accepted_dev, void *stream)
{
    if (!target_dev || !u_draw_dev || !out_dev || !accepted_dev || (n_draft > 0 && (!tokens_dev || !u_accept_dev)))
        SMX_FAIL(SMX_EINVAL, "smx_verify_draft: null argument");
    if (n_seq <= 0 || n_draft < 0 || n_draft > 65535 || vocab <= 0 || vocab > (1 << 24))
        SMX_FAIL(SMX_EINVAL, "smx_verify_draft: need n_seq >= 1, 0 <= n_draft <= 65535, 1 <= vocab <= 2^24");
    if (n_seq > kMaxBlocks / 4) SMX_FAIL(SMX_EUNSUPPORTED, "smx_verify_draft: too many sequences for one launch");
    if (target_stride < vocab || (draft_dev && n_draft > 0 && draft_stride < vocab))
        SMX_FAIL(SMX_EINVAL, "smx_verify_draft: rows must be at least vocab apart");
    if (((uintptr_t)target_dev | (uintptr_t)draft_dev) & 3) SMX_FAIL(SMX_EINVAL, "smx_verify_draft: misaligned pointer");
    SMX_HIP(launch_verify(target_dev, target_stride, n_draft > 0 ? draft_dev : nullptr, draft_stride, tokens_dev, lens_dev,
                          u_accept_dev, u_draw_dev, n_seq, n_draft, vocab, out_dev, accepted_dev, (hipStream_t)stream));
    return SMX_OK;
}

}  // extern "C"
