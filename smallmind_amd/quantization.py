"""Operator level of the backend: the IWeightTensor mirror and the per-op entry points.

Mirrors SmallMind.Quantization's operator boundary (IWeightTensor.cs:7-42): a weight knows its
Rows / Cols / Scheme, multiplies activations (`MatMul`, y = x W^T with k == Cols, n == Rows) and
dequantizes to fp32 (`ToFloat32`).  Dimension mismatches raise ValueError as the reference
raises ArgumentException (Q8WeightTensor.cs:43-48).

Device memory is held in torch tensors purely as allocation/stream plumbing; every computation
is a call into libsmx.so.
"""
from __future__ import annotations

import ctypes
from enum import IntEnum

import numpy as np

from . import _lib
from ._lib import SmxError, call


class GgufTensorType(IntEnum):
    """GGUF tensor type ids (GgufTensorType.cs:6-52) the backend implements, and SmallMind's own
    SMQ Q8Tensor / Q4Tensor blocks (1000 + QuantScheme id, QuantScheme.cs) in their upload
    layout (per 32 elements: the fp32 scale of their SMQ block, then the codes; smq_pack)."""
    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q8_0 = 8
    Q4_K = 12
    Q5_K = 13
    Q6_K = 14
    SMQ_Q8 = 1010
    SMQ_Q4 = 1011


BLOCK_ELEMS = {0: 1, 1: 1, 2: 32, 8: 32, 12: 256, 13: 256, 14: 256, 1010: 32, 1011: 32}
BLOCK_BYTES = {0: 4, 1: 2, 2: 18, 8: 34, 12: 144, 13: 176, 14: 210, 1010: 36, 1011: 20}


def smq_pack(qtype: int, data, scales, rows: int, cols: int, block_size: int) -> np.ndarray:
    """A Q8Tensor / Q4Tensor (codes as stored in an .smq file, fp32 scales per block_size
    elements of the flattened tensor) re-laid as SMX_TYPE_SMQ_Q8 / _Q4 upload bytes; no value
    changes (smx_smq_pack, host memory)."""
    d = np.ascontiguousarray(data).view(np.uint8).reshape(-1)
    sc = np.ascontiguousarray(scales, dtype=np.float32).reshape(-1)
    out = np.empty(rows * cols // 32 * BLOCK_BYTES[int(qtype)], np.uint8)
    call("smx_smq_pack", int(qtype), d.ctypes.data_as(ctypes.c_void_p), sc.ctypes.data_as(ctypes.c_void_p),
         rows, cols, block_size, out.ctypes.data_as(ctypes.c_void_p), out.size)
    return out


_T = None


def _torch():
    global _T
    if _T is None:
        import torch
        _T = torch
    return _T


def _ptr(t) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr())


def _stream():
    torch = _torch()
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _require_cuda(*ts):
    for t in ts:
        if not t.is_cuda:
            raise ValueError("operands must be device (cuda) tensors")
        if not t.is_contiguous():
            raise ValueError("operands must be contiguous")


def row_bytes(qtype: int, k: int) -> int:
    be = BLOCK_ELEMS[int(qtype)]
    if k % be:
        raise ValueError(f"row length {k} is not a multiple of the block size {be}")
    return k // be * BLOCK_BYTES[int(qtype)]


def dequantize(qtype: int, blocks, n: int):
    """GGUF blocks (device uint8 tensor) -> fp32 device tensor, bit-identical to
    GgufModelLoader.Convert*Tensor (GgufModelLoader.cs:419-917)."""
    torch = _torch()
    _require_cuda(blocks)
    out = torch.empty(n, dtype=torch.float32, device=blocks.device)
    call("smx_dequant", int(qtype), _ptr(blocks), n, _ptr(out), _stream())
    return out


def quantize(qtype: int, x):
    """fp32 device tensor -> GGUF blocks (device uint8 tensor) with the backend encoders."""
    torch = _torch()
    _require_cuda(x)
    n = x.numel()
    be = BLOCK_ELEMS[int(qtype)]
    if n % be:
        raise ValueError(f"{n} elements is not a multiple of the block size {be}")
    out = torch.empty(n // be * BLOCK_BYTES[int(qtype)], dtype=torch.uint8, device=x.device)
    call("smx_quantize", int(qtype), _ptr(x), n, _ptr(out), _stream())
    return out


def fill_normal(seed: int, n: int, std: float, device="cuda"):
    torch = _torch()
    out = torch.empty(n, dtype=torch.float32, device=device)
    call("smx_fill_normal", ctypes.c_uint64(seed), n, std, _ptr(out), _stream())
    return out


class GpuWeightTensor:
    """IWeightTensor backed by a repacked device weight (IWeightTensor.cs:7-42)."""

    def __init__(self, qtype: int, rows: int, cols: int, blocks):
        self._h = ctypes.c_void_p()
        if isinstance(blocks, np.ndarray) or isinstance(blocks, (bytes, bytearray)):
            buf = np.ascontiguousarray(np.frombuffer(blocks, np.uint8) if not isinstance(blocks, np.ndarray)
                                       else blocks.view(np.uint8).reshape(-1))
            if buf.size != rows * row_bytes(qtype, cols):
                raise ValueError("block buffer size does not match rows x cols")
            call("smx_weight_create", int(qtype), rows, cols, buf.ctypes.data_as(ctypes.c_void_p), 0,
                 ctypes.byref(self._h))
        else:
            _require_cuda(blocks)
            if blocks.numel() * blocks.element_size() != rows * row_bytes(qtype, cols):
                raise ValueError("block buffer size does not match rows x cols")
            _torch().cuda.synchronize()
            call("smx_weight_create", int(qtype), rows, cols, _ptr(blocks), 1, ctypes.byref(self._h))
        self.rows, self.cols, self.scheme = rows, cols, GgufTensorType(int(qtype))

    @property
    def Rows(self) -> int:
        return self.rows

    @property
    def Cols(self) -> int:
        return self.cols

    def mat_mul(self, activations, output, m: int, k: int, n: int):
        """IWeightTensor.MatMul: output[m][n] = activations[m][k] . W^T (k == Cols, n == Rows)."""
        _require_cuda(activations, output)
        if k != self.cols or n != self.rows:
            raise ValueError(f"k={k} must equal Cols={self.cols} and n={n} Rows={self.rows}")
        if activations.numel() < m * k or output.numel() < m * n:
            raise ValueError("activation/output buffers are too small")
        call("smx_weight_matmul", self._h, _ptr(activations), _ptr(output), m, k, n, _stream())
        return output

    def mat_mul_host(self, activations: np.ndarray, m: int, k: int, n: int, output: np.ndarray | None = None):
        """IWeightTensor.MatMul with host operands, as the reference takes them
        (ReadOnlySpan<float> activations, Span<float> output): numpy float32 arrays of at least
        m*k and m*n elements; synchronous (smx_weight_matmul_host)."""
        a = np.ascontiguousarray(activations, dtype=np.float32).reshape(-1)
        if output is None:
            output = np.empty((m, n), np.float32)
        if a.size < m * k or output.size < m * n or not output.flags.c_contiguous or output.dtype != np.float32:
            raise ValueError("activation/output buffers are too small or not contiguous float32")
        call("smx_weight_matmul_host", self._h, a.ctypes.data_as(ctypes.c_void_p),
             output.ctypes.data_as(ctypes.c_void_p), m, k, n)
        return output

    def to_float32_host(self) -> np.ndarray:
        """IWeightTensor.ToFloat32 into host memory: [Rows][Cols] float32 (smx_weight_to_float32_host)."""
        out = np.empty((self.rows, self.cols), np.float32)
        call("smx_weight_to_float32_host", self._h, out.ctypes.data_as(ctypes.c_void_p))
        return out

    def to_float32(self):
        """IWeightTensor.ToFloat32: [Rows][Cols] fp32 on the device."""
        torch = _torch()
        out = torch.empty((self.rows, self.cols), dtype=torch.float32, device="cuda")
        call("smx_weight_to_float32", self._h, _ptr(out), _stream())
        return out

    def close(self):
        if getattr(self, "_h", None) and self._h.value and _lib._lib is not None:
            _lib._lib.smx_weight_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        self.close()


# ---- elementwise / attention operators (device tensors) -----------------------------------------
def rmsnorm(x, gamma, eps: float = 1e-5):
    torch = _torch()
    _require_cuda(x, gamma)
    n = x.shape[-1]
    y = torch.empty_like(x)
    call("smx_rmsnorm", _ptr(x), _ptr(gamma), _ptr(y), x.numel() // n, n, eps, _stream())
    return y


def layernorm(x, gamma, beta, eps: float = 1e-5):
    torch = _torch()
    _require_cuda(x, gamma, beta)
    n = x.shape[-1]
    y = torch.empty_like(x)
    call("smx_layernorm", _ptr(x), _ptr(gamma), _ptr(beta), _ptr(y), x.numel() // n, n, eps, _stream())
    return y


def rope_tables(max_pos: int, head_dim: int, theta: float = 10000.0):
    c = np.empty((max_pos, head_dim // 2), np.float32)
    s = np.empty((max_pos, head_dim // 2), np.float32)
    call("smx_rope_tables", max_pos, head_dim, theta, c.ctypes.data_as(ctypes.c_void_p),
         s.ctypes.data_as(ctypes.c_void_p))
    return c, s


def rope_(data, pos0: int, cos_t, sin_t):
    """In place on data [heads][seq][hd]."""
    _require_cuda(data, cos_t, sin_t)
    h, s, hd = data.shape
    call("smx_rope", _ptr(data), h, s, hd, pos0, _ptr(cos_t), _ptr(sin_t), _stream())
    return data


def scale_mask_softmax_(scores, scale: float, cache_offset: int = 0):
    _require_cuda(scores)
    seq, kseq = scores.shape
    call("smx_scale_mask_softmax", _ptr(scores), scale, seq, kseq, cache_offset, _stream())
    return scores


def attention_decode(q, k_cache, v_cache, n_head: int, n_kv_head: int, head_dim: int,
                     ctx_stride: int, n_pos: int):
    torch = _torch()
    _require_cuda(q, k_cache, v_cache)
    out = torch.empty(n_head * head_dim, dtype=torch.float32, device=q.device)
    call("smx_attention_decode", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), n_head,
         n_kv_head, head_dim, ctx_stride, n_pos, _stream())
    return out


def attention_prefill(q, k_cache, v_cache, n_head: int, n_kv_head: int, head_dim: int,
                      ctx_stride: int, p_first: int, n_tok: int):
    torch = _torch()
    _require_cuda(q, k_cache, v_cache)
    out = torch.empty(n_tok * n_head * head_dim, dtype=torch.float32, device=q.device)
    call("smx_attention_prefill", _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), n_head,
         n_kv_head, head_dim, ctx_stride, p_first, n_tok, _stream())
    return out


def silu_mul(gate, up):
    torch = _torch()
    _require_cuda(gate, up)
    y = torch.empty_like(gate)
    call("smx_silu_mul", _ptr(gate), _ptr(up), _ptr(y), gate.numel(), _stream())
    return y


def gelu(x):
    torch = _torch()
    _require_cuda(x)
    y = torch.empty_like(x)
    call("smx_gelu", _ptr(x), _ptr(y), x.numel(), _stream())
    return y


def argmax(x) -> int:
    torch = _torch()
    _require_cuda(x)
    out = torch.empty(1, dtype=torch.int32, device=x.device)
    call("smx_argmax", _ptr(x), x.numel(), _ptr(out), _stream())
    return int(out.item())


def sample(logits, u: float, context=None, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
           min_p: float = 0.0, repetition_penalty: float = 1.0, presence_penalty: float = 0.0,
           frequency_penalty: float = 0.0, repetition_window: int = 0):
    """Next-token sampling in InferenceSession's order (InferenceSession.cs:565-606) on the
    device: (token, final probabilities).  logits and context (int32 token ids, oldest first)
    are cuda tensors; u in [0, 1) is the uniform draw (Random.NextDouble in the reference)."""
    torch = _torch()
    _require_cuda(logits)
    p = _lib.SamplingC(temperature, top_k, top_p, min_p, repetition_penalty, presence_penalty,
                       frequency_penalty, repetition_window)
    probs = torch.empty_like(logits)
    out = torch.empty(1, dtype=torch.int32, device=logits.device)
    n_ctx = 0 if context is None else context.numel()
    call("smx_sample", _ptr(logits), logits.numel(), _ptr(context) if n_ctx else None, n_ctx, ctypes.byref(p),
         float(u), _ptr(probs), _ptr(out), _stream())
    return int(out.item()), probs


# ---- serving operators: 8-bit KV cache, attention over it, drafted tokens ------------------------
# These are called once per layer and token, with kernels of a few microseconds: the checks below ask each
# tensor only what a wrong call would differ in, and sizes of work memory are kept per set of sizes.
def _raw_stream(index: int) -> int:
    torch = _torch()
    try:
        return torch._C._cuda_getCurrentRawStream(index)
    except AttributeError:
        return torch.cuda.current_stream(index).cuda_stream


class _Here:
    """The current device, already the right one."""

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        return False


_HERE = _Here()


def _on_device(index: int, *tensors):
    """Checks that the tensors are on cuda device `index` and makes it current (a context manager)."""
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"operands must be on cuda:{index}, not {t.device}")
    cuda = _torch().cuda
    return _HERE if cuda.current_device() == index else cuda.device(index)


def _c_int(n: int, what: str):
    """Refuses what a C int would take for another number."""
    if not -0x80000000 <= n <= 0x7FFFFFFF:
        raise ValueError(f"{what} {n} is out of range")


def _int32(t, n: int, what: str):
    if t.dtype is not _torch().int32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of {n} elements")


def _matrix_rows(t, width: int, what: str) -> int:
    """The distance between the rows of t [..., width], evenly spaced."""
    if t.is_contiguous() and t.dtype is _torch().float32:
        return width
    return _rows(t.unsqueeze(-2), 1, width, what)


def _rows(t, heads: int, head_dim: int, what: str) -> int:
    """The distance between the [heads][head_dim] rows of t [..., heads, head_dim], which may lie in the
    rows of a wider matrix (a fused projection)."""
    shape = t.shape
    if t.dtype is not _torch().float32 or len(shape) < 3 or shape[-2] != heads or shape[-1] != head_dim:
        raise ValueError(f"{what} must be float32 [..., {heads}, {head_dim}], is {t.dtype} {tuple(shape)}")
    row = heads * head_dim
    if t.is_contiguous() or t.numel() == 0:
        return row
    strides = t.stride()
    ok = (strides[-1] == 1 or head_dim == 1) and (strides[-2] == head_dim or heads == 1)
    step, n = None, 1
    for size, st in zip(reversed(shape[:-2]), reversed(strides[:-2])):
        if size == 1:
            continue
        if step is None:
            step = st
        elif st != n * step:
            ok = False
        n *= size
    step = row if step is None else step
    if not ok or step < row:
        raise ValueError(f"{what}: tokens must be evenly spaced rows of contiguous heads")
    return step


class GpuKvCache:
    """An 8-bit KV cache of n_slots sequences of up to ctx positions (smx_kv_cache_*): every row of
    head_dim values is kept as one Q8Tensor block, codes and an fp32 scale (Q8Tensor.cs:72-128).
    head_dim: a multiple of 8 up to 256.  Lives on `device` (default: the current one)."""

    def __init__(self, n_slots: int, n_kv_head: int, head_dim: int, ctx: int, device=None):
        self._h = ctypes.c_void_p()
        self._work = {}      # work memory of an attention call, by its sizes
        for n, what in ((n_slots, "n_slots"), (n_kv_head, "n_kv_head"), (head_dim, "head_dim"), (ctx, "ctx")):
            _c_int(n, what)
        torch = _torch()
        with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
            self.device = torch.device("cuda", torch.cuda.current_device())
            call("smx_kv_cache_create", n_slots, n_kv_head, head_dim, ctx, ctypes.byref(self._h))
        self.n_slots, self.n_kv_head, self.head_dim, self.ctx = n_slots, n_kv_head, head_dim, ctx

    @property
    def nbytes(self) -> int:
        b = ctypes.c_int64()
        call("smx_kv_cache_info", self._handle(), None, None, None, None, ctypes.byref(b))
        return b.value

    def append(self, k, v, slots, pos):
        """Writes token t's rows k[t], v[t] ([n_tok, n_kv_head, head_dim] float32, possibly slices of a fused
        projection) to position pos[t] of slot slots[t] (int32).  Places the cache does not have (-1) are
        skipped; a place named twice is left with undefined contents."""
        n, kv, hd, index = slots.numel(), self.n_kv_head, self.head_dim, self.device.index
        ks, vs = _rows(k, kv, hd, "k"), _rows(v, kv, hd, "v")
        if k.numel() != n * kv * hd or v.numel() != n * kv * hd:
            raise ValueError(f"k and v must hold one row per token ({n})")
        _int32(slots, n, "slots")
        _int32(pos, n, "pos")
        _c_int(n, "the number of tokens")
        with _on_device(index, k, v, slots, pos):
            if n:
                call("smx_kv_append", self._handle(), k.data_ptr(), ks, v.data_ptr(), vs, slots.data_ptr(),
                     pos.data_ptr(), n, _raw_stream(index))

    def read(self, slots, pos):
        """(k, v), each [n_tok, n_kv_head, head_dim] float32: the values the cache holds at these places (zeros
        at places it does not have)."""
        torch, n, index = _torch(), slots.numel(), self.device.index
        _int32(slots, n, "slots")
        _int32(pos, n, "pos")
        _c_int(n, "the number of tokens")
        with _on_device(index, slots, pos):
            k = torch.empty((n, self.n_kv_head, self.head_dim), dtype=torch.float32, device=self.device)
            v = torch.empty_like(k)
            if n:
                call("smx_kv_read", self._handle(), slots.data_ptr(), pos.data_ptr(), n, k.data_ptr(), v.data_ptr(),
                     _raw_stream(index))
        return k, v

    def _handle(self):
        if not self._h.value:
            raise ValueError("the cache is closed")
        return self._h

    def _work_bytes(self, n_seq: int, n_q: int, n_head: int, prefix_len: int, max_len: int) -> int:
        key = (n_seq, n_q, n_head, prefix_len, max_len)
        need = self._work.get(key)
        if need is None:
            b = ctypes.c_int64()
            call("smx_attention_work_bytes", self._handle(), *key, ctypes.byref(b))
            if len(self._work) >= 4096:
                self._work.clear()
            need = self._work[key] = b.value
        return need

    def close(self):
        if getattr(self, "_h", None) and self._h.value and _lib is not None and _lib._lib is not None:
            _lib._lib.smx_kv_cache_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        self.close()


def _attention_q8(q, cache, prefix, slots, lens, max_len, name):
    torch, h, index = _torch(), cache._handle(), cache.device.index
    if q.dim() != 4:
        raise ValueError("q must be [n_seq, n_q, n_head, head_dim]")
    n_seq, n_q, n_head, _ = q.shape
    stride = _rows(q, n_head, cache.head_dim, "q")
    if max_len is None:
        max_len = cache.ctx
    _c_int(max_len, "max_len")
    for n in prefix:
        _c_int(n, "prefix_slot or prefix_len")
    _c_int(n_seq * n_q * n_head, "n_seq * n_q * n_head")
    _int32(slots, n_seq, "slots")
    _int32(lens, n_seq, "lens")
    with _on_device(index, q, slots, lens):
        out = torch.empty(q.shape, dtype=torch.float32, device=cache.device)
        need = cache._work_bytes(n_seq, n_q, n_head, prefix[1] if prefix else 0, max_len)
        work = lens.new_empty((need,), dtype=torch.uint8) if need else None
        call(name, h, q.data_ptr(), stride, out.data_ptr(), n_seq, n_q, n_head, *prefix, slots.data_ptr(), lens.data_ptr(),
             max_len, work.data_ptr() if need else None, need, _raw_stream(index))
    return out


def attention_cached(q, cache: GpuKvCache, slots, lens, max_len: int | None = None):
    """Attention of the last n_q tokens of n_seq sequences over an 8-bit cache (smx_attention_cached).
    q [n_seq, n_q, n_head, head_dim] float32 (tokens may be rows of a fused projection); sequence b's
    positions are the first lens[b] of slot slots[b] (int32 on the device), its n_q tokens the last of them,
    each seeing all up to itself.  max_len: an upper bound of lens (default: ctx); a tight one is faster.
    Returns [n_seq, n_q, n_head, head_dim]; zeros for rows that see nothing and for slots the cache does not
    have."""
    return _attention_q8(q, cache, (), slots, lens, max_len, "smx_attention_cached")


def attention_shared(q, cache: GpuKvCache, prefix_slot: int, prefix_len: int, slots, lens, max_len: int | None = None):
    """attention_cached for sequences that all begin with the first prefix_len positions of slot prefix_slot,
    which are read once for all of them; slots and lens describe what each sequence has of its own, possibly
    nothing (smx_attention_shared)."""
    return _attention_q8(q, cache, (int(prefix_slot), int(prefix_len)), slots, lens, max_len, "smx_attention_shared")


def verify_draft(target, draft, tokens, u_accept, u_draw, lens=None):
    """Verification of drafted tokens (speculative decoding; smx_verify_draft).  target [n_seq, n_draft + 1,
    vocab] and draft [n_seq, n_draft, vocab]: the probabilities of the target and of the draft model (draft
    None: tokens chosen without a distribution); tokens [n_seq, n_draft] int32; u_accept [n_seq, n_draft] and
    u_draw [n_seq]: uniform numbers in [0, 1); lens [n_seq] int32: drafted tokens per sequence (default:
    n_draft, negative: an empty place).  Returns (out [n_seq, n_draft + 1], accepted [n_seq]) int32: the
    accepted tokens, one drawn token, then -1.  A token whose draft probability is NaN is refused, and not drawn in
    its place."""
    torch, index = _torch(), target.get_device()
    shape = target.shape
    if len(shape) != 3 or shape[1] < 1:
        raise ValueError("target must be [n_seq, n_draft + 1, vocab]")
    if index < 0:
        raise ValueError("operands must be device (cuda) tensors")
    n_seq, n_draft, vocab = shape[0], shape[1] - 1, shape[2]
    for n, what in ((n_seq, "n_seq"), (n_draft, "n_draft"), (vocab, "vocab")):
        _c_int(n, what)
    ts = _matrix_rows(target, vocab, "target")
    ds = 0
    if draft is not None:
        if draft.shape != (n_seq, n_draft, vocab):
            raise ValueError(f"draft must be {(n_seq, n_draft, vocab)}, is {tuple(draft.shape)}")
        ds = _matrix_rows(draft, vocab, "draft")
    for u, want, what in ((u_accept, (n_seq, n_draft), "u_accept"), (u_draw, (n_seq,), "u_draw")):
        if u.shape != want or u.dtype is not torch.float32 or not u.is_contiguous():
            raise ValueError(f"{what} must be contiguous float32 {want}")
    _int32(tokens, n_seq * n_draft, "tokens")
    if lens is not None:
        _int32(lens, n_seq, "lens")
    with _on_device(index, draft, tokens, u_accept, u_draw, lens):
        out = torch.empty((n_seq, n_draft + 1), dtype=torch.int32, device=target.device)
        accepted = torch.empty(n_seq, dtype=torch.int32, device=target.device)
        call("smx_verify_draft", target.data_ptr(), ts, None if draft is None else draft.data_ptr(), ds,
             tokens.data_ptr(), None if lens is None else lens.data_ptr(), u_accept.data_ptr(), u_draw.data_ptr(), n_seq,
             n_draft, vocab, out.data_ptr(), accepted.data_ptr(), _raw_stream(index))
    return out, accepted


# ---- serving operators over a paged KV cache ------------------------------------------------------
_ELEM = None


def _rows_like(t, dtype):
    """A contiguous tensor of t's shape and device (empty_like, the quickest way there, keeps strides)."""
    return _torch().empty_like(t) if dtype is t.dtype and t.is_contiguous() else t.new_empty(t.shape, dtype=dtype)


def _elem_type(dtype, what: str) -> int:
    """The smx_type of rows of this torch type."""
    global _ELEM
    if _ELEM is None:
        torch = _torch()
        _ELEM = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
    t = _ELEM.get(dtype)
    if t is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, is {dtype}")
    return t


def _token_rows(t, n_head, head_dim: int, what: str) -> int:
    """The distance between the [heads][head_dim] rows of t [n_tok, heads, head_dim], which may lie in the rows of a wider
    matrix (a fused projection)."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != head_dim or (n_head is not None and shape[1] != n_head):
        raise ValueError(f"{what} must be [n_tok, {n_head or 'heads'}, {head_dim}], is {tuple(shape)}")
    row = shape[1] * head_dim
    if t.is_contiguous() or t.numel() == 0:
        return row
    s = t.stride()
    step = s[0] if shape[0] > 1 else row
    if (s[2] != 1 and head_dim > 1) or (s[1] != head_dim and shape[1] > 1) or step < row:
        raise ValueError(f"{what}: tokens must be rows of contiguous heads")
    return step


def _floats(t, n: int, what: str):
    if t.dtype is not _torch().float32 or t.numel() != n or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous float32 tensor of {n} elements")


def _opt(t):
    return None if t is None else t.data_ptr()


class Rotation:
    """The rotation of queries and keys by position (smx_rotation).  cos and sin [n_pos, n_rot / 2] float32 on the device
    (rope_tables gives such); sections: how many pairs turn by each axis, in order (default: all by one); halves: pair j
    is channels j and j + n_rot / 2, otherwise 2 j and 2 j + 1."""

    def __init__(self, cos, sin, sections=None, halves: bool = False):
        if cos.dim() != 2 or cos.shape != sin.shape or cos.shape[0] < 1 or cos.shape[1] < 1:
            raise ValueError("cos and sin must be [n_pos, n_rot / 2]")
        n_pos, half = cos.shape
        _c_int(n_pos, "n_pos")
        _c_int(2 * half, "n_rot")
        _floats(cos, n_pos * half, "cos")
        _floats(sin, n_pos * half, "sin")
        sections = [half] if sections is None else [int(n) for n in sections]
        if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) != half:
            raise ValueError(f"sections must be 1 to 4 numbers that add up to {half}, are {sections}")
        self.cos, self.sin, self.n_axes = cos, sin, len(sections)
        self._c = _lib.RotationC(cos.data_ptr(), sin.data_ptr(), n_pos, 2 * half, int(bool(halves)), len(sections),
                                 (ctypes.c_int32 * 4)(*sections))


def _turning(rotation, pos, n: int):
    """(tables and positions to check, what the call takes for them)."""
    if rotation is None:
        return (), None, None
    if pos is None:
        raise ValueError("the rotation needs positions")
    _int32(pos, n * rotation.n_axes, "pos")
    return (rotation.cos, rotation.sin, pos), ctypes.byref(rotation._c), pos.data_ptr()


def _eps(eps: float) -> float:
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps {eps} must be finite and not negative")
    return eps


def qk_norm_rope(q, k, q_gamma=None, k_gamma=None, eps: float = 1e-6, rotation: Rotation | None = None, pos=None, dtype=None):
    """Norms of queries and keys for each head and the rotation by position in one pass (smx_qk_norm_rope).  q [n_tok, n_head,
    head_dim] and k [n_tok, n_kv_head, head_dim] float32, float16 or bfloat16 (tokens may be rows of a fused projection);
    gammas [head_dim] float32 (None: no norm); pos [n_tok], or [n_axes, n_tok], int32.  Returns (q, k) of `dtype` (default:
    as they come), rounded once."""
    index = q.get_device()
    if index < 0:
        raise ValueError("operands must be device (cuda) tensors")
    if q.dim() != 3 or k.dtype is not q.dtype or k.dim() != 3 or q.shape[0] != k.shape[0]:
        raise ValueError("q and k must be [n_tok, heads, head_dim] of one type")
    n, n_head, hd = q.shape
    qs, ks = _token_rows(q, n_head, hd, "q"), _token_rows(k, None, hd, "k")
    dtype = q.dtype if dtype is None else dtype
    tin, tout = _elem_type(q.dtype, "q"), _elem_type(dtype, "dtype")
    for g, what in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
        if g is not None:
            _floats(g, hd, what)
    for x, what in ((n, "n_tok"), (n_head, "n_head"), (k.shape[1], "n_kv_head"), (hd, "head_dim")):
        _c_int(x, what)
    turn, rot, at = _turning(rotation, pos, n)
    with _on_device(index, k, q_gamma, k_gamma, *turn):
        qo = _rows_like(q, dtype)
        ko = _rows_like(k, dtype)
        if n and n_head + k.shape[1]:
            call("smx_qk_norm_rope", tin, q.data_ptr(), qs, n_head, k.data_ptr(), ks, k.shape[1], hd, _opt(q_gamma), _opt(k_gamma),
                 _eps(eps), rot, at, n, tout, qo.data_ptr(), ko.data_ptr(), _raw_stream(index))
    return qo, ko


class GpuPagedCache:
    """A KV cache in pages of page_size positions (a power of two from 16 to 1024), float16 or bfloat16 (smx_paged_cache_*).  Position
    p of a sequence lies in page table[p // page_size], at place page * page_size + p % page_size of the cache; tables are
    the caller's.  head_dim: a multiple of 8 up to 256.  Lives on `device` (default: the current one)."""

    def __init__(self, dtype, n_pages: int, n_kv_head: int, head_dim: int, page_size: int = 64, device=None):
        self._h = ctypes.c_void_p()
        self._work = {}      # work memory of a call, by its sizes
        torch = _torch()
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"a paged cache is float16 or bfloat16, not {dtype}")
        for n, what in ((n_pages, "n_pages"), (n_kv_head, "n_kv_head"), (head_dim, "head_dim"), (page_size, "page_size")):
            _c_int(n, what)
        with torch.cuda.device(device if device is not None else torch.cuda.current_device()):
            self.device = torch.device("cuda", torch.cuda.current_device())
            call("smx_paged_cache_create", _elem_type(dtype, "dtype"), n_pages, n_kv_head, head_dim, page_size, ctypes.byref(self._h))
        self.dtype, self.n_pages, self.n_kv_head, self.head_dim, self.page_size = dtype, n_pages, n_kv_head, head_dim, page_size

    @property
    def nbytes(self) -> int:
        b = ctypes.c_int64()
        call("smx_paged_cache_info", self._handle(), None, None, None, None, None, ctypes.byref(b))
        return b.value

    def append(self, k, v, places, q=None, q_gamma=None, k_gamma=None, eps: float = 1e-6, rotation: Rotation | None = None, pos=None,
               dtype=None):
        """Writes token t's rows k[t], v[t] ([n_tok, n_kv_head, head_dim] float32, float16 or bfloat16, possibly slices of a fused
        projection) to place places[t] (int32; -1, or any that the cache does not have: skipped; one named twice is left
        with undefined contents).  With k_gamma or a rotation the keys are normed and turned as they are by qk_norm_rope; with q
        ([n_tok, n_head, head_dim] of k's type) so are the queries, and they are returned, of `dtype` (default: as they
        come)."""
        n, kv, hd, index = places.numel(), self.n_kv_head, self.head_dim, self.device.index
        ks, vs = _token_rows(k, kv, hd, "k"), _token_rows(v, kv, hd, "v")
        if k.shape[0] != n or v.shape[0] != n or v.dtype is not k.dtype:
            raise ValueError(f"k and v must hold one row per token ({n}), of one type")
        tin = tout = _elem_type(k.dtype, "k")
        _int32(places, n, "places")
        _c_int(n, "the number of tokens")
        n_head = qs = 0
        if q is not None:
            if q.dtype is not k.dtype or q.dim() != 3 or q.shape[0] != n or q.shape[1] < 1:
                raise ValueError(f"q must be [{n}, n_head, {hd}] of k's type")
            n_head, qs = q.shape[1], _token_rows(q, q.shape[1], hd, "q")
            _c_int(n_head, "n_head")
            dtype = q.dtype if dtype is None else dtype
            tout = _elem_type(dtype, "dtype")
        for g, what in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
            if g is not None:
                _floats(g, hd, what)
        turn, rot, at = _turning(rotation, pos, n)
        with _on_device(index, k, v, places, q, q_gamma, k_gamma, *turn):
            out = None if q is None else _rows_like(q, dtype)
            if n:
                call("smx_paged_append", self._handle(), tin, _opt(q), qs, n_head, k.data_ptr(), ks, v.data_ptr(), vs, _opt(q_gamma),
                     _opt(k_gamma), _eps(eps), rot, at, places.data_ptr(), n, tout, _opt(out), _raw_stream(index))
        return out

    def read(self, places):
        """(k, v), each [n_tok, n_kv_head, head_dim] of the cache's type: the rows at these places (zeros at places it does not
        have)."""
        torch, n, index = _torch(), places.numel(), self.device.index
        _int32(places, n, "places")
        _c_int(n, "the number of tokens")
        with _on_device(index, places):
            k = places.new_empty((n, self.n_kv_head, self.head_dim), dtype=self.dtype)
            v = torch.empty_like(k)
            if n:
                call("smx_paged_read", self._handle(), places.data_ptr(), n, k.data_ptr(), v.data_ptr(), _raw_stream(index))
        return k, v

    def evict(self, mass, lens, n_keep: int, n_recent: int, tables, new_tables):
        """Keeps n_keep positions of every sequence and KV head: the last n_recent and those others with the most weight in
        mass [n_seq, n_kv_head, max_len] float32 (the first of equals); all where there are no more.  lens [n_seq], tables
        [n_seq, pages] and new_tables [n_seq, pages] int32: the kept rows are copied in order to positions 0 .. of the new
        pages, which must be others than any sequence's old ones (smx_paged_evict).  Returns (kept [n_seq, n_kv_head, n_keep]
        int32, -1 beyond; new lens [n_seq] int32; their weights [n_seq, n_kv_head, n_keep] float32)."""
        index = self.device.index
        if mass.dim() != 3 or mass.shape[1] != self.n_kv_head or mass.shape[0] < 1:
            raise ValueError(f"mass must be [n_seq, {self.n_kv_head}, max_len]")
        n_seq, kv, max_len = mass.shape
        stride = _mass_rows(mass)
        _int32(lens, n_seq, "lens")
        for n, what in ((n_seq, "n_seq"), (max_len, "max_len"), (n_keep, "n_keep"), (n_recent, "n_recent")):
            _c_int(n, what)
        for t, what in ((tables, "tables"), (new_tables, "new_tables")):
            _table(t, n_seq, what)
        with _on_device(index, mass, lens, tables, new_tables):
            shape = (n_seq, kv, max(n_keep, 0))
            kept, new_lens, new_mass = lens.new_empty(shape), lens.new_empty((n_seq,)), mass.new_empty(shape)
            call("smx_paged_evict", self._handle(), mass.data_ptr(), stride, lens.data_ptr(), n_seq, max_len, n_keep, n_recent,
                 tables.data_ptr(), tables.shape[1], new_tables.data_ptr(), new_tables.shape[1], kept.data_ptr(),
                 new_lens.data_ptr(), new_mass.data_ptr(), _raw_stream(index))
        return kept, new_lens, new_mass

    def _handle(self):
        if not self._h.value:
            raise ValueError("the cache is closed")
        return self._h

    def _work_bytes(self, name: str, key, rules=()) -> int:
        need = self._work.get((name, key, rules))
        if need is None:
            b = ctypes.c_int64()
            extra = ()
            if name == "smx_attention_paged_work_bytes":
                c = _lib.AttentionRulesC(0.0, 0.0, None, None, rules[0], 0)
                extra = (ctypes.byref(c),)
            call(name, self._handle(), *key, *extra, ctypes.byref(b))
            if len(self._work) >= 4096:
                self._work.clear()
            need = self._work[(name, key, rules)] = b.value
        return need

    def close(self):
        if getattr(self, "_h", None) and self._h.value and _lib is not None and _lib._lib is not None:
            _lib._lib.smx_paged_cache_destroy(self._h)
            self._h = ctypes.c_void_p()

    def __del__(self):
        self.close()


def _table(t, n_seq: int, what: str):
    if t.dtype is not _torch().int32 or t.dim() != 2 or t.shape[0] != n_seq or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 [{n_seq}, pages] tensor")
    _c_int(t.shape[1], "pages")


def _mass_rows(mass) -> int:
    """The distance between the rows of mass [n_seq, n_kv_head, width], evenly spaced."""
    return _matrix_rows(mass, mass.shape[2], "mass")


def _rules(n_seq, n_head, scale, cap, slopes, window, prefix):
    if scale is None and cap == 0.0 and slopes is None and window == 0 and prefix is None:
        return None          # (what the C side takes for these)
    if slopes is not None:
        _floats(slopes, n_head, "slopes")
    if prefix is not None:
        _int32(prefix, n_seq, "prefix")
    _c_int(window, "window")
    for x, what in ((0.0 if scale is None else scale, "scale"), (cap, "cap")):
        if not 0.0 <= x < 3.4e38:
            raise ValueError(f"{what} {x} must be finite and not negative")
        if 0.0 < x < 1.4e-45:      # (0 in fp32, which stands for the default scale and for no cap)
            raise ValueError(f"{what} {x} is below the range of float32")
    if scale is not None and not scale > 0.0:
        raise ValueError("scale must be positive")
    return ctypes.byref(_lib.AttentionRulesC(0.0 if scale is None else scale, cap, _opt(slopes), _opt(prefix), window, 0))


def _paged_batch(q, cache, starts, lens, tables, max_q, max_len):
    """Checks what the calls over a batch have in common: (n_tok, n_head, n_seq, q's stride, q's type, max_len)."""
    if q.dim() != 3:
        raise ValueError("q must be [n_tok, n_head, head_dim]")
    n_tok, n_head, _ = q.shape
    stride = _token_rows(q, n_head, cache.head_dim, "q")
    t = _elem_type(q.dtype, "q")
    if t != _lib.F32 and q.dtype is not cache.dtype:
        raise ValueError(f"q must be float32 or the cache's {cache.dtype}, is {q.dtype}")
    n_seq = lens.numel()
    _int32(lens, n_seq, "lens")
    _int32(starts, n_seq + 1, "starts")
    _table(tables, n_seq, "tables")
    if max_len is None:
        max_len = min(tables.shape[1] * cache.page_size, 1 << 24)
    _c_int(max_q, "max_q")
    _c_int(max_len, "max_len")
    _c_int(n_tok * n_head, "n_tok * n_head")
    return n_tok, n_head, n_seq, stride, t, max_len


def attention_paged(q, cache: GpuPagedCache, starts, lens, tables, max_q: int, max_len: int | None = None, scale: float | None = None,
                    cap: float = 0.0, slopes=None, window: int = 0, prefix=None, lse: bool = False, out=None):
    """Attention of a ragged batch of new tokens over a paged cache (smx_attention_paged).  q [n_tok, n_head, head_dim] float32 or of the
    cache's type (tokens may be rows of a fused projection).  Sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1
    ([n_seq + 1]; at most max_q each) and the last of its lens[b] positions (already appended), which lie in the pages
    tables[b] ([n_seq, pages]); all int32 on the device.  max_len: an upper bound of lens (default: what the tables
    hold); a tight one is faster.  A token at position t sees positions p <= t; with window > 0, those with p > t - window; and the
    first prefix[b] ([n_seq] int32) whatever its own.  scale (default 1 / sqrt(head_dim)) times q . k, capped to cap *
    tanh(score / cap) where cap > 0, less slopes[h] * |t - p| ([n_head] float32).
    Returns [n_tok, n_head, head_dim] of q's type, or that and, with lse, the logarithms of the sums of exponentials
    [n_tok, n_head] float32.  Rows that see nothing are zeros (lse -inf).  Rows of no sequence are left as they are in
    `out`, undefined where that is not given.  `out` must not lie in q's memory."""
    torch, h, index = _torch(), cache._handle(), cache.device.index
    n_tok, n_head, n_seq, stride, t, max_len = _paged_batch(q, cache, starts, lens, tables, max_q, max_len)
    rules = _rules(n_seq, n_head, scale, cap, slopes, window, prefix)
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or not out.is_contiguous()):
        raise ValueError(f"out must be contiguous {q.dtype} {tuple(q.shape)}")
    with _on_device(index, q, starts, lens, tables, slopes, prefix, out):
        if out is None:
            out = _rows_like(q, q.dtype)
        sums = q.new_empty((n_tok, n_head), dtype=torch.float32) if lse else None
        need = cache._work_bytes("smx_attention_paged_work_bytes", (t, n_tok, n_head, n_seq, max_q, max_len), (window,))
        work = lens.new_empty((need,), dtype=torch.uint8) if need else None
        call("smx_attention_paged", h, t, q.data_ptr(), stride, out.data_ptr(), _opt(sums), n_tok, n_head, n_seq, starts.data_ptr(),
             lens.data_ptr(), tables.data_ptr(), tables.shape[1], max_q, max_len, rules, _opt(work), need, _raw_stream(index))
    return (out, sums) if lse else out


def attention_mass(q, lse, cache: GpuPagedCache, starts, lens, tables, max_q: int, max_len: int | None = None, mass=None,
                   scale: float | None = None, cap: float = 0.0, slopes=None, window: int = 0, prefix=None):
    """The attention weight that every position has received (smx_attention_mass): mass [n_seq, n_kv_head, width] float32 (None, or
    beyond width: 0) plus the sum over each sequence's new tokens and each KV head's query heads of exp(score - lse).  lse
    [n_tok, n_head] as attention_paged gives it for the same q, lengths and rules.  Returns [n_seq, n_kv_head, max_len]
    float32, 0 from lens[b] on: what evict decides by."""
    torch, h, index = _torch(), cache._handle(), cache.device.index
    n_tok, n_head, n_seq, stride, t, max_len = _paged_batch(q, cache, starts, lens, tables, max_q, max_len)
    rules = _rules(n_seq, n_head, scale, cap, slopes, window, prefix)
    _floats(lse, n_tok * n_head, "lse")
    width = mass_stride = 0
    if mass is not None:
        if mass.dim() != 3 or mass.shape[:2] != (n_seq, cache.n_kv_head):
            raise ValueError(f"mass must be [{n_seq}, {cache.n_kv_head}, width]")
        width, mass_stride = mass.shape[2], _mass_rows(mass)
        _c_int(width, "width")
    with _on_device(index, q, lse, starts, lens, tables, mass, slopes, prefix):
        out = lse.new_empty((n_seq, cache.n_kv_head, max(max_len, 0)))
        if out.numel() == 0 and max_len == 0:
            return out
        need = cache._work_bytes("smx_attention_mass_work_bytes", (t, n_head, n_seq, max_q, max_len))
        work = lens.new_empty((need,), dtype=torch.uint8) if need else None
        call("smx_attention_mass", h, t, q.data_ptr(), stride, lse.data_ptr(), _opt(mass), mass_stride, width, out.data_ptr(), n_tok,
             n_head, n_seq, starts.data_ptr(), lens.data_ptr(), tables.data_ptr(), tables.shape[1], max_q, max_len,
             rules, _opt(work), need, _raw_stream(index))
    return out


__all__ = ["GgufTensorType", "GpuWeightTensor", "SmxError", "dequantize", "quantize", "fill_normal",
           "rmsnorm", "layernorm", "rope_tables", "rope_", "scale_mask_softmax_", "attention_decode",
           "silu_mul", "gelu", "argmax", "sample", "row_bytes", "BLOCK_ELEMS", "BLOCK_BYTES", "GpuKvCache",
           "attention_cached", "attention_shared", "verify_draft", "Rotation", "qk_norm_rope", "GpuPagedCache",
           "attention_paged", "attention_mass"]
