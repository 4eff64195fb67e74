"""KV caches by handle: 16-bit or 8-bit rows, grouped heads, one length per slot, and attention over them, optionally behind a prefix
that all slots share (include/seedmi.h: seedmi_kv_append / seedmi_kv_read / seedmi_kv_attention).

``LlamaEngine`` keeps its static caches in 16 bits, one layout for all layers; these classes are the same caches for a serving loop of
its own: ``KVCache.new`` holds 1.03 bytes a value in the 8-bit block format ("mx8": e4m3 with one power-of-two scale per 32 values; a value
is off by up to 2^-4 of itself, the smallest of a block by more, 2.7 % rms) or two in the 16-bit one ("16"), ``KVCache.wrap`` takes tensors
that are there already (an engine's ``k_cache[i]`` / ``v_cache[i]`` among them).
A decode step is ``q = cache.append(qkv, cos, sin, lens, heads=H)`` and ``out = attention(q, lens + T)`` with an attention made once by
``KVAttention``; drafted chunks and prompt chunks are the same calls with more tokens per slot.

All calls are asynchronous on the current stream of the cache's device and allocate nothing but their outputs.  A ``KVAttention`` owns a
workspace: calls of one object belong on one stream (or need an event between them), and graphs that replay at the same time an object each.
"""
import ctypes as C
import math
from typing import Optional, Union

import torch

from . import lib as L

_FORMATS = {"16": L.KV_16BIT, "mx8": L.KV_MX8}
Lengths = Union[int, torch.Tensor]


# the raw stream of a device's current stream, without the Stream object around it (a decode step pays for every microsecond on the host)
_current_stream = torch._C._cuda_getCurrentRawStream


def _call(index, fn, name, lib, *args):
    """One library call on the current stream of device ``index``; the library launches on the current device, so that is switched to it
    for the call where the caller's is another."""
    prev = torch.cuda.current_device()
    if prev == index:
        rc = fn(*args, _current_stream(index))
    else:
        torch.cuda.set_device(index)
        try:
            rc = fn(*args, _current_stream(index))
        finally:
            torch.cuda.set_device(prev)
    if rc:
        L.check(rc, name, lib)


class KVCache:
    """Rows of keys and values, [slots, kv_heads, rows, head_dim] each; made by ``new`` or ``wrap``."""

    def __init__(self, k, v, k_scale, v_scale, dtype):
        fmt = "16" if k_scale is None else "mx8"
        if (k_scale is None) != (v_scale is None):
            raise ValueError("KVCache: scale bytes for both keys and values or for neither")
        if dtype not in (torch.bfloat16, torch.float16):
            raise L.SeedmiError(f"KVCache computes in bfloat16 or float16, not {dtype}")
        if k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"KVCache: keys {tuple(k.shape)} and values {tuple(v.shape)} must be [slots, kv_heads, rows, head_dim] alike")
        want = dtype if fmt == "16" else torch.uint8
        if k.dtype != want or v.dtype != want:
            raise ValueError(f"KVCache: a {fmt} cache of {dtype} holds {want}, not {k.dtype} / {v.dtype}")
        slots, heads, rows, dim = k.shape
        if dim not in (64, 128):
            raise L.SeedmiError(f"KVCache: head_dim {dim}: the kernels are built for 64 and 128")
        if min(slots, heads, rows) < 1:
            raise ValueError(f"KVCache: empty cache {tuple(k.shape)}")
        slot_rows, head_rows = self._row_strides(k, dim)
        if self._row_strides(v, dim) != (slot_rows, head_rows):
            raise ValueError("KVCache: keys and values must be laid out alike")
        if fmt == "mx8":
            for s in (k_scale, v_scale):
                if s.dtype != torch.uint8 or tuple(s.shape) != (slots, heads, rows, dim // 32):
                    raise ValueError(f"KVCache: scale bytes must be uint8 {(slots, heads, rows, dim // 32)}, not {s.dtype} {tuple(s.shape)}")
                if self._row_strides(s, dim // 32) != (slot_rows, head_rows):
                    raise ValueError("KVCache: scale bytes must be laid out like the rows they scale")
        for t in (v, k_scale, v_scale):
            if t is not None and t.device != k.device:
                raise ValueError("KVCache: tensors of more than one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.dtype, self.device, self.format = dtype, k.device, fmt
        self.slots, self.kv_heads, self.rows, self.head_dim = slots, heads, rows, dim
        if self.device.type != "cuda":
            raise L.SeedmiError("KVCache needs a HIP device (cuda:N); there is no CPU path")
        self.lib = L.load(dtype)
        p = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
        self.struct = L.KVCacheStruct(p(k), p(v), p(k_scale), p(v_scale), slot_rows, head_rows, slots, rows, heads, dim, _FORMATS[fmt])
        self._ref = C.byref(self.struct)
        self.index = self.device.index
        self._append, self._read = self.lib.seedmi_kv_append, self.lib.seedmi_kv_read

    @staticmethod
    def _row_strides(t, dim):
        """Strides of slots and heads in rows; a row is contiguous and rows follow each other."""
        ss, hs, rs, es = t.stride()
        ss, hs = (ss if t.shape[0] > 1 else t.shape[1] * t.shape[2] * dim), (hs if t.shape[1] > 1 else t.shape[2] * dim)
        if es != 1 or (rs != dim and t.shape[2] > 1) or ss % dim or hs % dim:
            raise ValueError(f"KVCache: rows must be contiguous and follow each other (strides {t.stride()})")
        return ss // dim, hs // dim

    @classmethod
    def new(cls, slots: int, kv_heads: int, rows: int, head_dim: int = 128, format: str = "mx8", dtype: torch.dtype = torch.bfloat16,
            device="cuda") -> "KVCache":
        """An empty cache.  ``dtype``: the 16-bit type of the queries, keys and values that go in and come out."""
        if format not in _FORMATS:
            raise ValueError(f"KVCache: format {format!r} (one of {sorted(_FORMATS)})")
        shape = (slots, kv_heads, rows, head_dim)
        if format == "16":
            k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
            return cls(k, v, None, None, dtype)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
        ks, vs = (torch.ones(shape[:3] + (head_dim // 32,), dtype=torch.uint8, device=device) for _ in range(2))
        return cls(k, v, ks, vs, dtype)

    @classmethod
    def wrap(cls, k: torch.Tensor, v: torch.Tensor, k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
             dtype: Optional[torch.dtype] = None) -> "KVCache":
        """A cache over tensors that exist: 16-bit rows, or e4m3 bytes (uint8) with their scale bytes and the 16-bit type to compute in."""
        return cls(k, v, k_scale, v_scale, dtype if dtype is not None else k.dtype)

    def slot(self, s: int) -> "KVCache":
        """One slot as a cache of its own (a prefix that others share, a prompt prefilled alone)."""
        cut = lambda t: None if t is None else t[s:s + 1]  # noqa: E731
        if not 0 <= s < self.slots:
            raise IndexError(f"KVCache: slot {s} of {self.slots}")
        return KVCache(self.k[s:s + 1], self.v[s:s + 1], cut(self.k_scale), cut(self.v_scale), self.dtype)

    def _lengths(self, what: str, n: Lengths, batch: int):
        """(host value, device pointer) of one length for all slots or of an int32 tensor with one each."""
        if isinstance(n, torch.Tensor):
            if n.dtype is not torch.int32 or n.get_device() != self.index or n.numel() < batch or not n.is_contiguous():
                raise ValueError(f"{what}: lengths must be a contiguous int32 tensor with one entry per slot on {self.device}")
            return 0, n.data_ptr()
        return L.int32(what, n), None

    def _rows_of(self, what: str, x: torch.Tensor, cols: int):
        """Row stride of x [rows, cols] in the cache's type on its device."""
        if x.dtype is self.dtype and x.get_device() == self.index and x.dim() == 2 and x.size(1) == cols and x.size(0) > 0:
            ld, one = x.stride()
            if one == 1:
                return ld if x.size(0) > 1 else cols
        raise ValueError(f"{what}: expected {self.dtype} rows of {cols} on {self.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")

    def _batch(self, what: str, rows: int, lens: Lengths, tokens: Optional[int]):
        """Slots of a call: ``rows`` query rows are ``tokens`` of each, by default of every slot that ``lens`` lists (or of all)."""
        if tokens is not None:
            if tokens < 1 or rows % tokens:
                raise ValueError(f"{what}: {rows} rows do not divide into slots of {tokens} tokens")
            batch = rows // tokens
        else:
            batch = lens.numel() if isinstance(lens, torch.Tensor) else self.slots
        if batch < 1 or batch > self.slots or rows % batch:
            raise ValueError(f"{what}: {rows} rows do not divide over {batch} of {self.slots} slots")
        return batch, rows // batch

    def append(self, qkv: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, past: Lengths, *, heads: int,
               pos_ids: Optional[torch.Tensor] = None, pos_base: int = 0, tokens: Optional[int] = None,
               q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """RoPE on the new rows' queries and keys, keys and values into the cache behind the ``past`` rows that each slot holds; returns the
        rotated queries [rows, heads * head_dim].  ``qkv`` [slots * T, (heads + 2 kv_heads) * head_dim] (q | k | v), slot-major, T = ``tokens``
        or, without it, what the rows divide into over the slots that ``past`` lists (all slots for an int); ``cos`` /
        ``sin`` [positions, head_dim] in the cache's type; positions are ``pos_ids`` (int64 [slots * T]) or pos_base + past + t."""
        D = self.head_dim
        heads, pos_base = L.int32("KVCache.append: heads", heads), L.int32("KVCache.append: pos_base", pos_base)
        ld = self._rows_of("KVCache.append", qkv, (heads + 2 * self.kv_heads) * D)
        B, T = self._batch("KVCache.append", qkv.shape[0], past, tokens)
        n, lens = self._lengths("KVCache.append: past", past, B)
        if not (cos.dtype is self.dtype and sin.dtype is self.dtype and cos.get_device() == self.index and sin.get_device() == self.index and
                cos.dim() == 2 and cos.shape == sin.shape and cos.size(1) == D and cos.is_contiguous() and sin.is_contiguous()):
            raise ValueError(f"KVCache.append: cos / sin must be contiguous {self.dtype} [positions, {D}] on {self.device}")
        pos = None
        if pos_ids is not None:
            if pos_ids.dtype is not torch.int64 or pos_ids.get_device() != self.index or pos_ids.numel() != B * T or not pos_ids.is_contiguous():
                raise ValueError(f"KVCache.append: pos_ids must be {B * T} contiguous int64 on {self.device}")
            pos = pos_ids.data_ptr()
        if q_out is None:
            q_out, ldq = torch.empty((B * T, heads * D), dtype=self.dtype, device=self.device), heads * D
        else:
            ldq = self._rows_of("KVCache.append (q_out)", q_out, heads * D)
            if q_out.size(0) != B * T:
                raise ValueError(f"KVCache.append: q_out has {q_out.size(0)} rows, not {B * T}")
        _call(self.index, self._append, "seedmi_kv_append", self.lib, self._ref, qkv.data_ptr(), ld, pos, pos_base, cos.data_ptr(), sin.data_ptr(),
              cos.size(0), q_out.data_ptr(), ldq, B, T, heads, n, lens)
        return q_out

    def read(self, start: Lengths, n: int, *, slots: Optional[int] = None, k_out: Optional[torch.Tensor] = None,
             v_out: Optional[torch.Tensor] = None):
        """Rows start .. start + n - 1 of every slot (or of the first ``slots``) of an mx8 cache as 16-bit (keys, values), [slots, kv_heads, n,
        head_dim].  Rows that a device-resident start puts outside the cache read as zeros."""
        B = slots if slots is not None else (start.numel() if isinstance(start, torch.Tensor) else self.slots)
        n = L.int32("KVCache.read: n", n)
        if not 1 <= B <= self.slots or n < 0:
            raise ValueError(f"KVCache.read: {n} rows of {B} of {self.slots} slots")
        at, starts = self._lengths("KVCache.read: start", start, B)
        shape = (B, self.kv_heads, n, self.head_dim)
        for t in (k_out, v_out):
            if t is not None and (tuple(t.shape) != shape or t.dtype is not self.dtype or t.get_device() != self.index or not t.is_contiguous()):
                raise ValueError(f"KVCache.read: outputs must be contiguous {self.dtype} {shape} on {self.device}")
        if k_out is None:
            k_out = torch.empty(shape, dtype=self.dtype, device=self.device)
        if v_out is None:
            v_out = torch.empty(shape, dtype=self.dtype, device=self.device)
        _call(self.index, self._read, "seedmi_kv_read", self.lib, self._ref, k_out.data_ptr(), v_out.data_ptr(), B, n, at, starts)
        return k_out, v_out


class LayerCaches:
    """One cache per decoder layer, alike in shape and format: what ``LlamaEngine.forward_kv`` appends to and attends over."""

    def __init__(self, caches):
        caches = list(caches)
        if not caches:
            raise ValueError("LayerCaches: no layers")
        first = caches[0]
        alike = lambda c: (c.slots, c.kv_heads, c.rows, c.head_dim, c.format, c.dtype, c.device)  # noqa: E731
        if any(alike(c) != alike(first) for c in caches):
            raise ValueError("LayerCaches: the layers' caches must be alike")
        self.layers = caches
        self.slots, self.rows, self.format, self.dtype, self.device = first.slots, first.rows, first.format, first.dtype, first.device
        self.array = (L.KVCacheStruct * len(caches))(*(c.struct for c in caches))

    def slot(self, s: int) -> "LayerCaches":
        """One slot of every layer (a shared prompt, a conversation prefilled alone)."""
        return LayerCaches(c.slot(s) for c in self.layers)


class KVAttention:
    """Attention of ``heads`` query heads over a ``KVCache``, ``tokens`` query rows per slot, made once and called every step.

    ``prefix`` / ``prefix_len``: rows 0 .. prefix_len - 1 of a one-slot cache in front of every slot's own rows, seen whole by every query.
    ``kv_max``: the longest slot expected (default: the cache's rows); it decides how keys are split over workgroups, never the result's
    definition.  ``causal``: query t of T sees its slot's rows up to its own; False: all of them (the keys of an encoder).  The object owns
    its workspace: calls that may run at the same time (two streams, two graphs) need an object each.  It is made outside of graph captures
    and called inside or outside of them."""

    def __init__(self, cache: KVCache, heads: int, tokens: int = 1, slots: Optional[int] = None, kv_max: int = 0,
                 prefix: Optional[KVCache] = None, prefix_len: int = 0, scale: Optional[float] = None, causal: bool = True):
        if prefix is None and prefix_len:
            raise ValueError("KVAttention: prefix_len without a prefix")
        if prefix is not None and (prefix.dtype != cache.dtype or prefix.device != cache.device):
            raise ValueError("KVAttention: prefix and cache must have one type and one device")
        if heads < 1 or heads % cache.kv_heads or tokens < 1:
            raise ValueError(f"KVAttention: {heads} query heads on {cache.kv_heads} key heads, {tokens} tokens")
        heads, tokens = L.int32("KVAttention: heads", heads), L.int32("KVAttention: tokens", tokens)
        self.cache, self.prefix, self.prefix_len = cache, prefix, L.int32("KVAttention: prefix_len", prefix_len)
        self.heads, self.tokens, self.slots = heads, tokens, cache.slots if slots is None else slots
        if not 1 <= self.slots <= cache.slots:
            raise ValueError(f"KVAttention: {self.slots} of {cache.slots} slots")
        self.kv_max, self.causal = L.int32("KVAttention: kv_max", kv_max), 1 if causal else 0
        self.scale = 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale)
        self._pref = self.prefix._ref if self.prefix_len else None
        need = cache.lib.seedmi_kv_attention_workspace_bytes(cache._ref, self.slots, tokens, heads, self.kv_max, self.prefix_len)
        with torch.cuda.device(cache.index):
            if need and torch.cuda.is_current_stream_capturing():
                # (a capture records the initialisation and does not run it: calls before the first replay would join on whatever is there)
                raise L.SeedmiError("KVAttention: this one needs a workspace, which a stream that captures a graph cannot initialise: make the "
                                    "object before the capture")
        self.workspace = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
        if need:
            _call(cache.index, cache.lib.seedmi_kv_attention_workspace_init, "seedmi_kv_attention_workspace_init", cache.lib,
                  self.workspace.data_ptr(), need)
            torch.cuda.current_stream(cache.device).synchronize()                  # ready for a first call on any stream
        self._home = _current_stream(cache.index)
        self._ws = (self.workspace.data_ptr(), need) if need else (None, 0)
        self._fn, self._rows, self._cols = cache.lib.seedmi_kv_attention, self.slots * tokens, heads * cache.head_dim

    def __call__(self, q: torch.Tensor, kv_len: Lengths, out: Optional[torch.Tensor] = None, plus: int = 0) -> torch.Tensor:
        """q [slots * tokens, heads * head_dim] -> out of the same shape; ``kv_len``: rows each slot holds, the query rows' own included: an
        int of 0 or more, or an int32 tensor with one entry per slot, 0 or less for an idle one.  ``plus`` is added to an int and to a tensor's
        entries that are not negative: ``attention(q, past, plus=T)`` takes the lengths that ``append`` took.  Queries that see nothing get
        zeros."""
        c, cols, rows = self.cache, self._cols, self._rows
        ldq = c._rows_of("KVAttention", q, cols)
        if q.size(0) != rows:
            raise ValueError(f"KVAttention: {q.size(0)} query rows, made for {self.slots} slots of {self.tokens}")
        n, lens = c._lengths("KVAttention: kv_len", kv_len, self.slots)
        if plus:
            n = L.int32("KVAttention: kv_len + plus", n + plus)
        if out is None:
            out, ldo = torch.empty((rows, cols), dtype=c.dtype, device=c.device), cols
        else:
            ldo = c._rows_of("KVAttention (out)", out, cols)
            if out.size(0) != rows:
                raise ValueError(f"KVAttention: out has {out.size(0)} rows, not {rows}")
        if self.workspace is not None and _current_stream(c.index) != self._home:
            self.workspace.record_stream(torch.cuda.current_stream(c.device))      # (freed memory is not handed on while that stream uses it)
        _call(c.index, self._fn, "seedmi_kv_attention", c.lib, c._ref, self._pref, self.prefix_len, q.data_ptr(), ldq, out.data_ptr(), ldo, self.slots,
              self.tokens, self.heads, n, lens, self.kv_max, self.scale, self.causal, self._ws[0], self._ws[1])
        return out
