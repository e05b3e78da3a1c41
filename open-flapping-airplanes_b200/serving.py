"""Serving operators over a paged key/value cache, on the current stream of their tensors' device: the torch view of the "serving over a
paged cache" part of include/ofa_b200.h, which says what each computes.

    cache = KVCache.empty(n_pages, page_size, n_kv_heads, head_dim, "e4m3")     # one per layer
    batch = KVBatch(q_start, kv_len, pages, max_new=..., max_kv=...)            # one per step, shared by the layers
    kv_append(cache, batch, k, v)                                               # this step's keys and values to their pages
    o = paged_attention(cache, batch, q)                                        # this step's queries over them
    k, v = kv_read(cache, batch, n_rows)                                        # cached rows back as bf16
    logits_process(logits, tokens=..., repetition=..., mask=..., out=logits)    # penalties, biases, a grammar's mask

Nothing is copied, cast or made contiguous behind the caller's back: a tensor of another type, device or layout than an operator takes is refused with an
OfaError. No call waits for the device or reads from it, and results carry no gradient. Index tensors are int32 and are read by the kernels, so a captured graph sees what they hold when it
is replayed.
"""
import ctypes as C
import importlib.util
import math

import torch

from . import capi
from .build import host_path
from .tasks import OfaError

E4M3 = torch.float8_e4m3fn
_TYPES = {"bf16": torch.bfloat16, "e4m3": E4M3}
_INT_MAX = 2 ** 31 - 1                                        # ctypes cuts what is larger to 32 bits without a word
BAD_PAGE, BAD_LENGTH, BAD_ROWS, TIMEOUT = 1, 2, 4, 8          # bits of a batch's status word


def _refuse(msg):
    raise OfaError(capi.BAD_ARGUMENT, msg)


def _want(name, t, dtype, shape, device, inner=True):
    """A CUDA tensor of this type and shape (None: any size) on `device` (None: any), its last axis dense."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        _refuse(f"{name} has to be a CUDA tensor")
    if t.dtype != dtype:
        _refuse(f"{name} has to be {dtype}, not {t.dtype}")
    s = t.shape
    if len(s) != len(shape) or any(w is not None and w != n for w, n in zip(shape, s)):
        _refuse(f"{name} has shape {tuple(s)}, not {tuple('any' if w is None else w for w in shape)}")
    if max(s, default=0) > _INT_MAX:
        _refuse(f"{name} has shape {tuple(s)}: at most 2^31 - 1 along an axis")
    if device is not None and t.device != device:
        _refuse(f"{name} is on {t.device}, not on {device}")
    if inner and len(s) and s[-1] > 1 and t.stride(-1) != 1:
        _refuse(f"the last axis of {name} has to be dense")


# The current stream's handle and the current device, without an object around them (0.1 instead of 1.2 us a call)
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_BF16, _F32, _I32 = torch.bfloat16, torch.float32, torch.int32


def _call(fn, index, *args):
    """fn(*args, current stream of device `index`), with that device current."""
    if _current() == index:
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream(index))
    if rc:
        raise OfaError(rc, _lib().ofa_serving_last_error().decode())


_loaded = None


def _lib():
    global _loaded
    if _loaded is None:
        _loaded = capi.load()
    return _loaded


def _bind():
    """The extension that build.build_host() compiled for this torch, bound to the loaded library; None where there is none. Its functions return results, the code of an entry point that
    refused, or None for arguments that are not plainly right: the code below then finds out what is wrong with them."""
    spec = importlib.util.spec_from_file_location("_serving", host_path(torch.__version__))
    try:
        _serving = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(_serving)
    except ImportError:
        return None
    lib = _lib()
    addr = lambda f: C.cast(f, C.c_void_p).value  # noqa: E731
    _serving.bind(addr(lib.ofa_kv_append), addr(lib.ofa_kv_read), addr(lib.ofa_paged_attention), addr(lib.ofa_paged_attention_workspace), addr(lib.ofa_logits_process))
    return _serving


_fast_module = ()


def _fast():
    global _fast_module
    if _fast_module == ():
        _fast_module = _bind()
    return _fast_module


def _done(rc):
    if rc:
        raise OfaError(rc, _lib().ofa_serving_last_error().decode())


def _rows(name, t, shape, cache):
    """The strides of bf16 rows [n_rows, heads, head_dim] on the cache's device; what is wrong with them otherwise."""
    try:
        if t.dtype is _BF16 and t.get_device() == cache.index and (shape is None or t.shape == shape) and t.shape[0] <= _INT_MAX:
            s = t.stride()
            if len(s) == 3 and s[2] == 1 and t.shape[2] == cache.head_dim:
                return s
    except AttributeError:
        pass
    _want(name, t, _BF16, (None, None, cache.head_dim) if shape is None else shape, cache.device)
    return t.stride()                                           # a last axis of one element, any stride


def _array(name, t, dtype, rows, index, device):
    """A dense [rows] array's address."""
    try:
        if t.dtype is dtype and t.get_device() == index and t.shape == (rows,) and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    _want(name, t, dtype, (rows,), device)
    return t.data_ptr()


def _table(name, t, dtype, shape, index, device):
    """(address, row stride) of a [rows, n] array with dense rows"""
    try:
        if t.dtype is dtype and t.get_device() == index:
            s = t.stride()
            if len(s) == 2 and s[1] == 1 and t.shape[0] == shape[0] and (shape[1] is None or t.shape[1] == shape[1]) and max(t.shape) <= _INT_MAX:
                return t.data_ptr(), s[0]
    except AttributeError:
        pass
    _want(name, t, dtype, shape, device)
    return t.data_ptr(), t.stride(0)


class KVCache:
    """Pages of keys and values: k and v [n_pages, n_kv_heads, page_size, head_dim], bf16 or float8_e4m3fn, any strides that keep rows on 16-byte
    boundaries and are the same for both; for e4m3 also k_scale and v_scale [n_pages, n_kv_heads, page_size], uint8. The tensors stay the caller's."""

    def __init__(self, k, v, k_scale=None, v_scale=None):
        e4m3 = isinstance(k, torch.Tensor) and k.dtype == E4M3
        _want("k", k, E4M3 if e4m3 else torch.bfloat16, (None,) * 4, None)
        _want("v", v, k.dtype, k.shape, k.device)
        if k.stride() != v.stride():
            _refuse(f"k and v have different strides: {k.stride()} and {v.stride()}")
        if e4m3:
            _want("k_scale", k_scale, torch.uint8, k.shape[:3], k.device, inner=False)
            _want("v_scale", v_scale, torch.uint8, k.shape[:3], k.device, inner=False)
            if k_scale.stride() != v_scale.stride():
                _refuse("k_scale and v_scale have different strides")
        elif k_scale is not None or v_scale is not None:
            _refuse("a bf16 cache has no scales")
        self.k, self.v, self.k_scale, self.v_scale, self.device, self.index = k, v, k_scale, v_scale, k.device, k.get_device()
        self.n_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        if self.head_dim not in (64, 128):
            _refuse(f"head_dim {self.head_dim}: 64 and 128 are built")
        self.scale = 1.0 / math.sqrt(self.head_dim)
        c = self.c = capi.KvCache()
        c.dtype, c.head_dim, c.n_kv_heads, c.page_size, c.n_pages = capi.KV_E4M3 if e4m3 else capi.KV_BF16, self.head_dim, self.n_kv_heads, self.page_size, self.n_pages
        c.k, c.v = k.data_ptr(), v.data_ptr()
        c.page_stride, c.head_stride, c.row_stride = k.stride()[:3]
        if e4m3:
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.scale_page_stride, c.scale_head_stride, c.scale_row_stride = k_scale.stride()
        self.ref, self.address = C.byref(c), C.addressof(c)

    @classmethod
    def empty(cls, n_pages, page_size, n_kv_heads, head_dim, dtype="bf16", device="cuda"):
        """A cache of its own; its rows are zeros."""
        if dtype not in _TYPES:
            _refuse(f"cache dtype {dtype!r} is neither 'bf16' nor 'e4m3'")
        make = lambda *s, t: torch.zeros(s, dtype=t, device=device)  # noqa: E731
        shape = (n_pages, n_kv_heads, page_size)
        scales = [make(*shape, t=torch.uint8) for _ in range(2)] if dtype == "e4m3" else []
        return cls(make(*shape, head_dim, t=_TYPES[dtype]), make(*shape, head_dim, t=_TYPES[dtype]), *scales)


class KVBatch:
    """The sequences of a step: q_start [n_seqs + 1], kv_len [n_seqs], pages [n_seqs, max_pages], int32 on the device. max_new and max_kv: the longest chunk
    and context as far as the program knows them; they choose how the work is cut, not what is computed. status: an int32 tensor whose first element
    collects BAD_PAGE, BAD_LENGTH, BAD_ROWS and TIMEOUT."""

    def __init__(self, q_start, kv_len, pages, max_new=0, max_kv=0, status=None):
        _want("pages", pages, torch.int32, (None, None), None)
        n = pages.shape[0]
        _want("kv_len", kv_len, torch.int32, (n,), pages.device)
        _want("q_start", q_start, torch.int32, (n + 1,), pages.device)
        if status is not None:
            _want("status", status, torch.int32, (None,), pages.device)
            if not status.numel():
                _refuse("status is empty")
        if max_new < 0 or max_kv < 0:
            _refuse(f"max_new {max_new}, max_kv {max_kv}")
        self.q_start, self.kv_len, self.pages, self.status, self.device, self.index = q_start, kv_len, pages, status, pages.device, pages.get_device()
        c = self.c = capi.KvBatch()
        c.n_seqs, c.max_pages, c.pages_stride = n, pages.shape[1], pages.stride(0)
        c.q_start, c.kv_len, c.pages = q_start.data_ptr(), kv_len.data_ptr(), pages.data_ptr()
        c.max_new, c.max_kv = min(max_new, _INT_MAX), min(max_kv, _INT_MAX)
        c.status = status.data_ptr() if status is not None else None
        self.ref, self.address = C.byref(c), C.addressof(c)


def _same_device(cache, batch):
    if cache.index != batch.index:
        _refuse(f"the cache is on {cache.device}, the batch on {batch.device}")


def _move(read, cache, batch, k, v, n_rows):
    _same_device(cache, batch)
    f = _fast()
    if f is not None:
        got = f.move(read, cache.address, batch.address, cache.index, -1 if n_rows is None else n_rows, k, v)
        if got is not None:
            return _done(got) if type(got) is int else got
    fn = _lib().ofa_kv_read if read else _lib().ofa_kv_append
    rows = k.shape[0] if n_rows is None and isinstance(k, torch.Tensor) and k.dim() else n_rows
    shape = (rows, cache.n_kv_heads, cache.head_dim)
    if k is None and read:
        k, v = torch.empty(shape, dtype=_BF16, device=cache.device), torch.empty(shape, dtype=_BF16, device=cache.device)
    a, b = _rows("k", k, shape, cache), _rows("v", v, shape, cache)
    _call(fn, cache.index, cache.ref, batch.ref, k.data_ptr(), v.data_ptr(), shape[0], a[0], a[1], b[0], b[1])
    return k, v


def kv_append(cache, batch, k, v):
    """Rows k and v [n_rows, n_kv_heads, head_dim] (bf16; views of a fused projection will do) to their pages, in the cache's type."""
    _move(False, cache, batch, k, v, None)


def kv_read(cache, batch, n_rows=None, k=None, v=None):
    """The batch's n_rows rows out of their pages, as bf16 [n_rows, n_kv_heads, head_dim] pairs (written into k and v where these are given)."""
    if k is None or v is None:
        if n_rows is None or n_rows < 0 or k is not None or v is not None:
            _refuse("kv_read needs n_rows, or k and v to write to")
        return _move(True, cache, batch, None, None, n_rows)
    _move(True, cache, batch, k, v, n_rows)
    return k, v


def paged_attention(cache, batch, q, out=None, scale=None, causal=True, window=0, with_lse=False):
    """Attention of q [n_rows, n_heads, head_dim] (bf16) over the batch's pages; scale: 1/sqrt(head_dim) by default. Returns out, of q's shape, or with
    with_lse (out, lse [n_rows, n_heads] fp32). Rows that no sequence brings are left as they were."""
    _same_device(cache, batch)
    scale = cache.scale if scale is None else scale
    f = _fast()
    if f is not None:
        got = f.attend(cache.address, batch.address, cache.index, q, out, scale, causal, window, with_lse)
        if got is not None:
            return _done(got) if type(got) is int else got
    window = max(-1, min(window, _INT_MAX))                      # as wide as that: wider than any context
    sq = _rows("q", q, None, cache)
    n_rows, n_heads, _ = q.shape
    if out is None:
        out = torch.empty_like(q, requires_grad=False)
    so = _rows("out", out, q.shape, cache)
    lse = torch.empty((n_rows, n_heads), dtype=_F32, device=cache.device) if with_lse else None
    need = _lib().ofa_paged_attention_workspace(cache.ref, batch.ref, n_rows, n_heads)
    # from torch's allocator: a graph that captures the call keeps its own
    work = torch.empty((need,), dtype=torch.uint8, device=cache.device) if need else None
    a = capi.PagedAttentionArgs(n_rows, n_heads, q.data_ptr(), sq[0], sq[1], out.data_ptr(), so[0], so[1], lse.data_ptr() if with_lse else None, scale, bool(causal), window,
                                work.data_ptr() if need else None, need)
    _call(_lib().ofa_paged_attention, cache.index, cache.ref, batch.ref, C.byref(a))
    return (out, lse) if with_lse else out


def logits_process(logits, tokens=None, n_tokens=None, n_prompt=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, mask=None, out=None):
    """Penalties of repeated tokens, biases and a bit mask on logits [n_rows, vocab] (bf16 or fp32); returns out (a new tensor by default; out=logits works in place).
    tokens [n_rows, max_tokens], n_tokens, n_prompt [n_rows], bias_ids [n_rows, n] and mask [n_rows, ceil(vocab / 32)] are int32, the rest fp32."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in (_F32, _BF16):
        _refuse("logits have to be a bf16 or fp32 tensor")
    f = _fast()
    if f is not None:
        got = f.process(logits, out, tokens, n_tokens, n_prompt, repetition, presence, frequency, bias_ids, bias, mask)
        if got is not None:
            return _done(got) if type(got) is int else got
    kind, dev, index = logits.dtype, logits.device, logits.get_device()
    if index < 0 or logits.dim() != 2:
        _want("logits", logits, kind, (None, None), None)
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty_like(logits, requires_grad=False)
    src, src_row = _table("logits", logits, kind, (rows, vocab), index, dev)
    dst, dst_row = _table("out", out, kind, (rows, vocab), index, dev)
    text = text_row = most = made = first = ids = bias_row = n_bias = weight = words = words_row = 0
    if tokens is not None:
        text, text_row = _table("tokens", tokens, _I32, (rows, None), index, dev)
        most = tokens.shape[1]
        made = 0 if n_tokens is None else _array("n_tokens", n_tokens, _I32, rows, index, dev)
        first = 0 if n_prompt is None else _array("n_prompt", n_prompt, _I32, rows, index, dev)
    elif not (n_tokens is n_prompt is repetition is presence is frequency is None):
        _refuse("penalties and token counts need tokens")
    rep = 0 if repetition is None else _array("repetition", repetition, _F32, rows, index, dev)
    pres = 0 if presence is None else _array("presence", presence, _F32, rows, index, dev)
    freq = 0 if frequency is None else _array("frequency", frequency, _F32, rows, index, dev)
    if (bias_ids is None) != (bias is None):
        _refuse("bias_ids and bias come together")
    if bias is not None:
        ids, row = _table("bias_ids", bias_ids, _I32, (rows, None), index, dev)
        n_bias = bias_ids.shape[1]
        weight, bias_row = _table("bias", bias, _F32, (rows, n_bias), index, dev)
        if bias_row != row and rows > 1:
            _refuse("bias and bias_ids have different strides")
    if mask is not None:
        words, words_row = _table("mask", mask, _I32, (rows, (vocab + 31) // 32), index, dev)
    a = capi.LogitsArgs(capi.DTYPE_F32 if kind is _F32 else capi.DTYPE_BF16, rows, vocab, src, src_row, dst, dst_row, text, text_row, most, made, first, rep, pres, freq,
                        ids, weight, bias_row, n_bias, words, words_row)
    _call(_lib().ofa_logits_process, index, C.byref(a))
    return out
