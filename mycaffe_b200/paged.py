"""Paged key/value cache and the per-head norm with rotation, over the C ABI (``mca_paged_*``, ``mca_qk_norm_rope_*``).

``PagedCache`` holds the pages of one layer; a ``PagedBatch`` describes a step's new tokens, which may be prompts, chunks of
prompts and single tokens together.  A layer's step is ``append`` (norm and rotation of queries and keys, keys and values into
their pages) and ``attend``.  ``QkNormRope`` is the norm and rotation itself; its ``forward`` and ``backward`` are the form for
training.  The reference has neither: its decode takes one token of one sequence over a contiguous cache
(CudaExtension.llm32.llama2/Files/llama2_gpu.cpp:32-111).

Calls are enqueued on the current stream of the tensors' device and may be captured into CUDA graphs.  torch is used for device
memory and streams only.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from . import function_ids as ids


class McaHeads(C.Structure):
    _fields_ = [("data", C.c_void_p), ("stride_b", C.c_int64), ("stride_t", C.c_int64), ("stride_h", C.c_int64)]


class McaQkRotation(C.Structure):
    _fields_ = [("q_weight", C.c_void_p), ("k_weight", C.c_void_p), ("cos_table", C.c_void_p), ("sin_table", C.c_void_p),
                ("table_len", C.c_int), ("flags", C.c_int), ("eps", C.c_float)]


class McaPagedCache(C.Structure):
    _fields_ = [("k_pages", C.c_void_p), ("v_pages", C.c_void_p), ("page_stride", C.c_int64)] + [
        (n, C.c_int) for n in ("n_pages", "page_size", "n_heads", "n_kv_heads", "head_size", "dtype")] + [("status", C.c_void_p)]


class McaPagedBatch(C.Structure):
    _fields_ = [("starts", C.c_void_p), ("lengths", C.c_void_p), ("page_table", C.c_void_p)] + [
        (n, C.c_int) for n in ("table_stride", "n_seqs", "n_tokens", "max_new", "max_len")]


STATUS_WORDS = 8

_DTYPES = {torch.float32: ids.MCA_DTYPE_F32, torch.bfloat16: ids.MCA_DTYPE_BF16}


class PagedError(RuntimeError):
    def __init__(self, code, what):
        super().__init__(f"{what} failed with {code}")
        self.code = int(code)


def _dtype(t, what):
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what}: float32 or bfloat16 is wanted, got {t.dtype}")
    return _DTYPES[t.dtype]


def _heads(t, what, shape, dtype, device, written=False):
    """A (..., heads, head_size) tensor as the C side sees it; rows of heads are read, or written, where they lie."""
    s = t.stride()
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise ValueError(f"{what}: {tuple(shape)} of {dtype} on {device} is wanted, got {tuple(t.shape)} of {t.dtype} on {t.device}")
    if s[-1] != 1:
        raise ValueError(f"{what}: a head's elements have to be contiguous")
    if written and 0 in s and any(step == 0 and n > 1 for step, n in zip(s, t.shape)):
        raise ValueError(f"{what}: an expanded tensor's rows lie on one another and cannot be written")
    return McaHeads(t.data_ptr(), s[0] if len(s) == 4 else 0, s[-3], s[-2])


def _indices(t, what, shape, device):
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what}: contiguous int32 of shape {shape} on {device} is wanted")
    return t.data_ptr()


def _vector(t, what, size, device):
    if t is None:
        return None
    if t.dtype != torch.float32 or t.device != device or not t.is_contiguous() or t.numel() != size:
        raise ValueError(f"{what}: {size} contiguous float32 on {device} are wanted")
    return t.data_ptr()


# the current stream's handle; without building a Stream object where torch offers that
_stream_handle = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(device, name, function, *args):
    """``function(*args, stream)`` with the device current, on its current stream."""
    index = device.index
    if torch.cuda.current_device() == index:
        rc = function(*args, _stream_handle(index))
    else:
        with torch.cuda.device(device):
            rc = function(*args, _stream_handle(index))
    if rc:
        raise PagedError(rc, name)


class QkNormRope:
    """Norm of each head and rotation by position: y = R(position) (w * x / sqrt(mean(x^2) + eps)).

    cos, sin: (positions, head_size / 2) float32 (``mca_rope_tables_host``), or None: no rotation.  halves: pair p is
    (x[p], x[p + head_size / 2]), else (x[2p], x[2p + 1]) as the reference's rope.  norm False: the rotation alone."""

    def __init__(self, cos, sin, q_weight=None, k_weight=None, eps=1e-5, norm=True, halves=False):
        self._lib = _lib.load()
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if not norm:
            q_weight = k_weight = None
        self._keep = (cos, sin, q_weight, k_weight)   # the C side holds addresses
        some = next((t for t in self._keep if t is not None), None)
        self.device = None if some is None else some.device
        self.head_size = None
        if cos is not None:
            if cos.dim() != 2:
                raise ValueError("cos: (positions, head_size / 2) is wanted")
            self.head_size = 2 * cos.shape[1]
            _vector(sin, "sin", cos.numel(), self.device)
        for w in (q_weight, k_weight):
            if w is not None and self.head_size is None:
                self.head_size = w.numel()
        self.norm = bool(norm)
        self.weights = (q_weight is not None, k_weight is not None)
        self.c = McaQkRotation(_vector(q_weight, "q_weight", self.head_size, self.device), _vector(k_weight, "k_weight", self.head_size, self.device),
                               None if cos is None else _vector(cos, "cos", cos.numel(), self.device), None if sin is None else sin.data_ptr(),
                               0 if cos is None else cos.shape[0], (ids.MCA_QK_NORM if norm else 0) | (ids.MCA_ROPE_HALVES if halves else 0), float(eps))

    def check(self, head_size, device):
        if self.head_size not in (None, head_size):
            raise ValueError(f"tables and weights are for a head size of {self.head_size}, not {head_size}")
        if self.device not in (None, device):
            raise ValueError(f"tables and weights are on {self.device}, not on {device}")

    def _common(self, q, k, positions):
        if q.dim() != 4:
            raise ValueError("q: (B, T, heads, head_size) is wanted")
        B, T, H, D = q.shape
        KV = 0 if k is None else k.shape[2]
        self.check(D, q.device)
        dt = _dtype(q, "q")
        pos = None if positions is None else _indices(positions, "positions", (B, T), q.device)
        return B, T, H, KV, D, dt, pos

    def forward(self, q, k, q_out, k_out, positions=None):
        """q (B,T,heads,D) and k (B,T,kv_heads,D) -> q_out, k_out of the same shapes; any strides but the last (transposed views of
        (B,heads,T,D) tensors, parts of a packed projection).  k and k_out may be None."""
        B, T, H, KV, D, dt, pos = self._common(q, k, positions)
        dev, qs, ks = q.device, (B, T, H, D), (B, T, KV, D)
        a = [_heads(q, "q", qs, q.dtype, dev), _heads(q_out, "q_out", qs, q.dtype, dev, True)]
        b = [None, None] if k is None else [C.byref(_heads(k, "k", ks, q.dtype, dev)), C.byref(_heads(k_out, "k_out", ks, q.dtype, dev, True))]
        _call(dev, "mca_qk_norm_rope_forward", self._lib.mca_qk_norm_rope_forward, C.byref(self.c), C.byref(a[0]), b[0], pos, dt, B, T, H, KV, D,
              C.byref(a[1]), b[1])

    def backward(self, q, k, dq_out, dk_out, dq, dk, positions=None, weight_grads=True):
        """From the forward's inputs and the gradients of its outputs: fills dq, dk and returns (dq_weight, dk_weight), float32,
        None for a weight that there is not (or with ``weight_grads`` False)."""
        B, T, H, KV, D, dt, pos = self._common(q, k, positions)
        dev, qs, ks = q.device, (B, T, H, D), (B, T, KV, D)
        a = [C.byref(_heads(t, n, qs, q.dtype, dev, t is dq)) for t, n in ((q, "q"), (dq_out, "dq_out"), (dq, "dq"))]
        b = [None] * 3 if k is None else [C.byref(_heads(t, n, ks, q.dtype, dev, t is dk)) for t, n in ((k, "k"), (dk_out, "dk_out"), (dk, "dk"))]
        want = (weight_grads and self.weights[0], weight_grads and self.weights[1] and k is not None)
        dw = [torch.empty(D, device=dev) if w else None for w in want]
        need = self._lib.mca_qk_norm_rope_backward_scratch_floats(D) if any(want) else 0
        scratch = torch.empty(need, device=dev) if need > 0 else None
        ptr = [None if t is None else t.data_ptr() for t in dw]
        _call(dev, "mca_qk_norm_rope_backward", self._lib.mca_qk_norm_rope_backward, C.byref(self.c), a[0], b[0], pos, a[1], b[1], dt, B, T, H,
              KV, D, a[2], b[2], ptr[0], ptr[1], None if scratch is None else scratch.data_ptr(), max(need, 0))
        return tuple(dw)


class PagedBatch:
    """A step's new tokens (see ``PagedCache.batch``)."""

    def __init__(self, c, n_tokens, device, keep):
        self.c, self.ref, self.n_tokens, self.device, self._keep = c, C.byref(c), n_tokens, device, keep


class PagedCache:
    """The pages of one layer: k_pages, v_pages (n_pages, page_size, kv_heads, head_size), float32 or bfloat16; pages may lie apart
    (a slice of a larger pool).  status: STATUS_WORDS int32 zeros on the device, 16-byte aligned, where the calls over this cache record what
    they refuse; None: the device's own words, which all such caches and ``QkNormRope`` share."""

    def __init__(self, k_pages, v_pages, n_heads, status=None):
        self._lib = _lib.load()
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
            raise ValueError("k_pages and v_pages: two alike tensors (n_pages, page_size, kv_heads, head_size) are wanted")
        n_pages, page, kv, hs = k_pages.shape
        if k_pages.stride() != v_pages.stride() or k_pages.stride()[1:] != (kv * hs, hs, 1):
            raise ValueError("k_pages and v_pages: contiguous within a page, with the same distance between pages")
        if status is not None:
            _indices(status, "status", (STATUS_WORDS,), k_pages.device)
        self._keep = (k_pages, v_pages, status)
        self.device, self.n_heads, self.kv_heads, self.head_size, self.page_size = k_pages.device, int(n_heads), kv, hs, page
        self.c = McaPagedCache(k_pages.data_ptr(), v_pages.data_ptr(), k_pages.stride(0), n_pages, page, self.n_heads, kv, hs, _dtype(k_pages, "k_pages"),
                              None if status is None else status.data_ptr())
        self._ref = C.byref(self.c)

    def batch(self, starts, lengths, page_table, n_tokens, max_new, max_len):
        """The new tokens of sequence b are rows [starts[b], starts[b + 1]) of the token tensors and the last of its lengths[b]
        positions; page_table[b, i] is the page of positions [i page_size, (i + 1) page_size), -1 where it is not held.  All int32 on
        the device.  n_tokens: rows of the token tensors; max_new, max_len: upper bounds of the new tokens and of the positions of a
        sequence."""
        n, stride, dev = lengths.shape[0], page_table.shape[-1], self.device
        c = McaPagedBatch(_indices(starts, "starts", (n + 1,), dev), _indices(lengths, "lengths", (n,), dev),
                          _indices(page_table, "page_table", (n, stride), dev), stride, n, n_tokens, max_new, max_len)
        return PagedBatch(c, n_tokens, dev, (starts, lengths, page_table))

    def _device_of(self, batch):
        if batch.device is not self.device and batch.device != self.device:   # a batch of this cache has this cache's own object
            raise ValueError(f"batch: its arrays are on {batch.device}, the pages on {self.device}")
        return self.device

    def append(self, batch, rotation, q, k, v, q_out):
        """Norm and rotation of the new tokens' q into q_out and of k into the pages; v into its pages.  q, q_out (n_tokens, heads,
        head_size), k, v (n_tokens, kv_heads, head_size)."""
        n, dev = batch.n_tokens, self._device_of(batch)
        rotation.check(self.head_size, dev)
        dt, qs, ks = _dtype(q, "q"), (n, self.n_heads, self.head_size), (n, self.kv_heads, self.head_size)
        a = (_heads(q, "q", qs, q.dtype, dev), _heads(k, "k", ks, q.dtype, dev), _heads(v, "v", ks, q.dtype, dev),
             _heads(q_out, "q_out", qs, q.dtype, dev, True))
        _call(dev, "mca_paged_append", self._lib.mca_paged_append, self._ref, batch.ref, C.byref(rotation.c), dt, C.byref(a[0]), C.byref(a[1]),
              C.byref(a[2]), C.byref(a[3]))

    def attend(self, batch, q, out, scale=None):
        """out = attention of the new tokens' q over their sequences' pages (their own keys among them); both (n_tokens, heads,
        head_size), and out not overlapping q or the pages.  scale: positive; None: 1 / sqrt(head_size)."""
        if scale is not None and not scale > 0.0:   # the C side's zero is its default
            raise ValueError(f"scale: a positive number or None is wanted, got {scale}")
        dev, shape = self._device_of(batch), (batch.n_tokens, self.n_heads, self.head_size)
        dt = _dtype(q, "q")
        a, o = _heads(q, "q", shape, q.dtype, dev), _heads(out, "out", shape, q.dtype, dev, True)
        need = self._lib.mca_paged_attention_workspace_bytes(self._ref, batch.ref, dt)
        # of the current stream's allocator (or a captured graph's own pool): no two calls that overlap share it
        work = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
        _call(dev, "mca_paged_attention", self._lib.mca_paged_attention, self._ref, batch.ref, dt, C.byref(a), scale or 0.0, C.byref(o),
              None if work is None else work.data_ptr(), max(need, 0))

    def status(self):
        """What the calls over this cache refused since the last time this was asked -- of a cache without status words of its own, what those
        of all such callers on the device did: (kind, detail, detail, how many), all zero if nothing.  Waits for the device."""
        torch.cuda.synchronize(self.device)
        st = (C.c_int * 4)()
        with torch.cuda.device(self.device):
            rc = self._lib.mca_paged_status_of(self.c.status, st) if self.c.status else self._lib.mca_paged_status(st)
        if rc:
            raise PagedError(rc, "mca_paged_status")
        return tuple(st)
