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
        work = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
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


__all__ = ["GgufTensorType", "GpuWeightTensor", "SmxError", "dequantize", "quantize", "fill_normal",
           "rmsnorm", "layernorm", "rope_tables", "rope_", "scale_mask_softmax_", "attention_decode",
           "silu_mul", "gelu", "argmax", "sample", "row_bytes", "BLOCK_ELEMS", "BLOCK_BYTES", "GpuKvCache",
           "attention_cached", "attention_shared", "verify_draft"]
