"""KV caches for long contexts over the C ABI: fp16 or 4-bit rows, attention with capped or biased scores and document or
prefix masks, accumulated attention weights and eviction by them (kcb_cache_* in include/kernelcore_b200.h)."""
from __future__ import annotations

import ctypes as C

import torch

from . import lib

BLOCK = 32  # channels that share a scale and a minimum in the 4-bit format


class _Cache(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("bits", "n_seqs", "kv_heads", "head_dim", "capacity")] + [("k", C.c_void_p), ("v", C.c_void_p)] + [
        (n, C.c_int64) for n in ("k_row", "k_head", "k_seq", "v_row", "v_head", "v_seq")] + [
        (n, C.c_void_p) for n in ("n_keys", "next_pos", "positions", "weights")]


class _Attn(C.Structure):
    _fields_ = [("n_tokens", C.c_int), ("heads", C.c_int), ("scale", C.c_float), ("softcap", C.c_float), ("max_bias", C.c_float), ("causal", C.c_int),
                ("accumulate", C.c_int)] + [(n, C.c_void_p) for n in ("prefix", "q_pos", "q_doc", "k_doc", "mask")] + [
        (n, C.c_int64) for n in ("mask_token", "mask_seq", "q_token", "q_head", "q_seq", "out_token", "out_head", "out_seq")]


_L = lib.raw
_L.kcb_cache_bytes.restype = C.c_size_t
_L.kcb_cache_bytes.argtypes = [C.c_int] * 5
_L.kcb_cache_append.argtypes = [C.POINTER(_Cache), C.c_void_p, C.c_void_p, C.c_int, C.c_int64, C.c_int64, C.c_void_p]
_L.kcb_cache_read.argtypes = [C.POINTER(_Cache), C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p]
_L.kcb_cache_evict_workspace_bytes.restype = C.c_size_t
_L.kcb_cache_evict_workspace_bytes.argtypes = [C.POINTER(_Cache), C.c_int]
_L.kcb_cache_evict.argtypes = [C.POINTER(_Cache), C.c_int, C.c_int, C.c_void_p, C.c_size_t, C.c_void_p]
_L.kcb_cache_attention_workspace_bytes.restype = C.c_size_t
_L.kcb_cache_attention_workspace_bytes.argtypes = [C.POINTER(_Cache), C.POINTER(_Attn)]
_L.kcb_cache_attention.argtypes = [C.POINTER(_Cache), C.POINTER(_Attn), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]


_stream = torch._C._cuda_getCurrentRawStream  # of a device index; the tensor-free form of torch.cuda.current_stream


def _launch(fn, device: torch.device, *args) -> None:
    """fn(*args, stream) with the tensors' device current, on the stream that is current there."""
    if torch.cuda.current_device() == device.index:
        status = fn(*args, _stream(device.index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _stream(device.index))
    if status:
        lib.check(status, fn.__name__)


def _used_here(t: torch.Tensor, home: int) -> None:
    """A workspace of stream `home` that went to the current stream: its memory is not given away while that still runs."""
    if _stream(t.device.index) != home:
        t.record_stream(torch.cuda.current_stream(t.device))


def _on(t: torch.Tensor, dtype, shape, what: str, device) -> int:
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{what}: a contiguous {dtype} tensor of shape {tuple(shape)} on {device} is needed, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def cache_bytes(bits: int, n_seqs: int, kv_heads: int, head_dim: int, capacity: int) -> int:
    return _L.kcb_cache_bytes(bits, n_seqs, kv_heads, head_dim, capacity)


class KVCache:
    """The buffers of a cache and the counts beside them.  16 bits: k and v are fp16 [n_seqs][capacity][kv_heads][head_dim]
    (any strides whose innermost is 1).  4 bits: k and v are uint8 of cache_bytes(...) in all.  The tensors are the
    caller's; the object keeps references to them."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, *, kv_heads: int, head_dim: int, capacity: int, bits: int = 16, n_keys: torch.Tensor | None = None,
                 next_pos: torch.Tensor | None = None, positions: torch.Tensor | None = None, weights: torch.Tensor | None = None):
        if k.device.type != "cuda" or v.device != k.device:
            raise ValueError(f"k and v must be on one CUDA device, got {k.device} and {v.device}")
        c = _Cache(bits=bits, kv_heads=kv_heads, head_dim=head_dim, capacity=capacity)
        self.device = k.device
        if bits == 16:
            for name, t in (("k", k), ("v", v)):
                if t.dtype != torch.float16 or t.dim() != 4 or tuple(t.shape[1:]) != (capacity, kv_heads, head_dim) or t.shape[0] != k.shape[0] or t.stride(3) != 1:
                    raise ValueError(f"{name}: fp16 [n_seqs][{capacity}][{kv_heads}][{head_dim}] with contiguous rows is needed, got {t.dtype} {tuple(t.shape)}")
            c.n_seqs = k.shape[0]
            c.k_seq, c.k_row, c.k_head = k.stride()[:3]
            c.v_seq, c.v_row, c.v_head = v.stride()[:3]
        else:
            one = cache_bytes(bits, 1, kv_heads, head_dim, capacity)
            if not one or k.dtype != torch.uint8 or not k.is_contiguous() or k.numel() % one or v.dtype != torch.uint8 or v.numel() != k.numel() or not v.is_contiguous():
                raise ValueError(f"k and v: contiguous uint8 buffers of {one} bytes per sequence are needed, got {k.dtype} {tuple(k.shape)}, {v.dtype} {tuple(v.shape)}")
            c.n_seqs = k.numel() // one
        c.k, c.v = k.data_ptr(), v.data_ptr()
        for name, t, dtype, shape in (("n_keys", n_keys, torch.int32, (c.n_seqs,)), ("next_pos", next_pos, torch.int32, (c.n_seqs,)),
                                      ("positions", positions, torch.int32, (c.n_seqs, kv_heads, capacity)),
                                      ("weights", weights, torch.float32, (c.n_seqs, kv_heads, capacity))):
            if t is not None:
                setattr(c, name, _on(t, dtype, shape, name, self.device))
        self.k, self.v, self.n_keys, self.next_pos, self.positions, self.weights = k, v, n_keys, next_pos, positions, weights
        self.bits, self.n_seqs, self.kv_heads, self.head_dim, self.capacity = bits, c.n_seqs, kv_heads, head_dim, capacity
        self.struct, self._ref = c, C.byref(c)
        self._evict_ws: dict[int, tuple] = {}  # by `keep`, kept: captured graphs go on using theirs

    @classmethod
    def empty(cls, n_seqs: int, kv_heads: int, head_dim: int, capacity: int, bits: int = 16, evictable: bool = False, device="cuda") -> "KVCache":
        """A cache without rows.  evictable: with positions and attention weights beside the rows."""
        device = torch.device(device)
        if device.type == "cuda" and device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        if bits == 16:
            k, v = (torch.zeros(n_seqs, capacity, kv_heads, head_dim, dtype=torch.float16, device=device) for _ in range(2))
        else:
            k, v = (torch.zeros(n_seqs, cache_bytes(bits, 1, kv_heads, head_dim, capacity), dtype=torch.uint8, device=device) for _ in range(2))
        n, p = (torch.zeros(n_seqs, dtype=torch.int32, device=device) for _ in range(2))
        pos = torch.zeros(n_seqs, kv_heads, capacity, dtype=torch.int32, device=device) if evictable else None
        w = torch.zeros(n_seqs, kv_heads, capacity, device=device) if evictable else None
        return cls(k, v, kv_heads=kv_heads, head_dim=head_dim, capacity=capacity, bits=bits, n_keys=n, next_pos=p, positions=pos, weights=w)

    def append(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """New rows behind those in use: fp32 [n_seqs][n_tokens][kv_heads][head_dim], heads and channels contiguous, k and v
        with the same strides (slices of one q|k|v product are)."""
        shape, stride = k.shape, k.stride()
        if len(shape) != 4 or shape[0] != self.n_seqs or shape[2] != self.kv_heads or shape[3] != self.head_dim or stride[3] != 1 or v.shape != shape or \
                v.stride() != stride or (self.kv_heads > 1 and stride[2] != self.head_dim) or k.dtype != torch.float32 or v.dtype != torch.float32 or \
                k.device != self.device or v.device != self.device:
            raise ValueError(f"k, v: fp32 [{self.n_seqs}][n_tokens][{self.kv_heads}][{self.head_dim}] on {self.device} with the same strides are needed, got " +
                             " and ".join(f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}" for t in (k, v)))
        if shape[1] and shape[0]:
            _launch(_L.kcb_cache_append, self.device, self._ref, k.data_ptr(), v.data_ptr(), shape[1], stride[1], stride[0])

    def read(self, first: int, count: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Slots first .. first + count - 1 as fp32 [n_seqs][count][kv_heads][head_dim], zeros where no row is in use."""
        if first < 0 or count < 0 or first + count > self.capacity:
            raise ValueError(f"slots {first} .. {first + count - 1} of {self.capacity}")
        k, v = (torch.empty(self.n_seqs, count, self.kv_heads, self.head_dim, device=self.device) for _ in range(2))
        if k.numel():
            _launch(_L.kcb_cache_read, self.device, self._ref, first, count, k.data_ptr(), v.data_ptr())
        return k, v

    def evict(self, keep: int, recent: int) -> None:
        """Sequences that hold more than `keep` rows drop the least attended ones (never one of the `recent` newest tokens)."""
        ws = self._evict_ws.get(keep)
        if ws is None:
            n = max(16, _L.kcb_cache_evict_workspace_bytes(self._ref, keep))
            buf = torch.empty(n, dtype=torch.uint8, device=self.device)
            ws = self._evict_ws[keep] = (buf, buf.data_ptr(), n, _stream(self.device.index))
        if self.n_seqs:
            _launch(_L.kcb_cache_evict, self.device, self._ref, keep, recent, ws[1], ws[2])
            _used_here(ws[0], ws[3])


class Attention:
    """Attention of n_tokens query tokens per sequence over a cache, with the masks given here; holds the workspace, so two
    calls of one object must not run at the same time, and which a graph that captured a call goes on using.  What the masks contain may change between calls."""

    def __init__(self, cache: KVCache, *, n_tokens: int, heads: int, scale: float | None = None, softcap: float = 0.0, max_bias: float = 0.0, causal: bool = True,
                 prefix: torch.Tensor | None = None, q_pos: torch.Tensor | None = None, q_doc: torch.Tensor | None = None, k_doc: torch.Tensor | None = None,
                 mask: torch.Tensor | None = None, accumulate: bool = False):
        S, dev = cache.n_seqs, cache.device
        a = _Attn(n_tokens=n_tokens, heads=heads, scale=cache.head_dim ** -0.5 if scale is None else scale, softcap=softcap, max_bias=max_bias,
                  causal=int(causal), accumulate=int(accumulate))
        for name, t, shape in (("prefix", prefix, (S,)), ("q_pos", q_pos, (S, n_tokens)), ("q_doc", q_doc, (S, n_tokens)), ("k_doc", k_doc, (S, cache.capacity))):
            if t is not None:
                setattr(a, name, _on(t, torch.int32, shape, name, dev))
        if mask is not None:
            if mask.dtype != torch.float16 or mask.dim() != 3 or mask.shape[0] != S or mask.shape[1] != n_tokens or mask.shape[2] < cache.capacity or \
                    mask.stride(2) != 1 or mask.device != dev:
                raise ValueError(f"mask: fp16 [{S}][{n_tokens}][{cache.capacity} or more] with contiguous rows is needed, got {mask.dtype} {tuple(mask.shape)}")
            a.mask, a.mask_seq, a.mask_token = mask.data_ptr(), mask.stride(0), mask.stride(1)
        self.cache, self.struct, self._ref = cache, a, C.byref(a)
        self._keep = (prefix, q_pos, q_doc, k_doc, mask)
        self.shape = torch.Size((S, n_tokens, heads, cache.head_dim))
        self._empty, self._strides = self.shape.numel() == 0, None
        n = _L.kcb_cache_attention_workspace_bytes(cache._ref, self._ref)
        self.workspace = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        self._ws = (self.workspace.data_ptr(), n) if n else (None, 0)
        self._home = _stream(dev.index)

    def __call__(self, q: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """q: fp32 [n_seqs][n_tokens][heads][head_dim] (contiguous channels, any other strides); out likewise, not overlapping q."""
        dev = self.cache.device
        if out is None:
            out = torch.empty(self.shape, device=dev)
        qs, os = q.stride(), out.stride()
        if q.shape != self.shape or out.shape != self.shape or q.dtype != torch.float32 or out.dtype != torch.float32 or qs[3] != 1 or os[3] != 1 or \
                q.device != dev or out.device != dev:
            raise ValueError(f"q, out: fp32 {tuple(self.shape)} with contiguous channels on {dev} are needed, got " +
                             " and ".join(f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}" for t in (q, out)))
        if self._strides != (qs, os):
            a = self.struct
            a.q_seq, a.q_token, a.q_head, _ = qs
            a.out_seq, a.out_token, a.out_head, _ = os
            self._strides = (qs, os)
        if self._empty:
            return out
        _launch(_L.kcb_cache_attention, dev, self.cache._ref, self._ref, q.data_ptr(), out.data_ptr(), *self._ws)
        if self.workspace is not None:
            _used_here(self.workspace, self._home)
        return out
