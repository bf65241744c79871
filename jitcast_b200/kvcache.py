"""A paged key/value cache on the GPU, and attention over it: the serving form of a layer's time attention.

The forwards recompute a series' whole context on every call. A caller that forecasts again and again as patches
arrive keeps each layer's keys and values instead: ``PagedCache.append`` stores a step's new tokens (rotating
keys and queries on the way), ``PagedCache.attention`` runs their attention over everything cached, with a sliding
window and sinks, and ``PagedCache.read`` returns cached tokens. The cache holds 16-bit values, or 4-bit codes with
a scale and a minimum per 32 dims. All run on torch CUDA tensors, enqueued on torch's current stream, through
``jc_kv_*`` of ``include/jitcast_b200.h`` (which defines formats and semantics).
"""

from __future__ import annotations

import ctypes
import math

from . import _lib
from ._lib import BF16, FP16, c_int, c_ll, c_vp, check

__all__ = ["PagedCache", "Step", "rope_table"]

GROUP = 32  # dims that share a 4-bit row's (scale, min)


class _Cache(ctypes.Structure):
    """jc_kv_cache"""

    _fields_ = [("bits", c_int), ("pages", c_int), ("page_size", c_int), ("kv_heads", c_int), ("head_dim", c_int),
                ("k", c_vp), ("v", c_vp), ("k_scale", c_vp), ("v_scale", c_vp)]


class _Step(ctypes.Structure):
    """jc_kv_step"""

    _fields_ = [("sequences", c_int), ("tokens", c_int), ("max_new", c_int), ("max_length", c_int), ("start", c_vp),
                ("length", c_vp), ("page_table", c_vp), ("table_pages", c_int), ("ld_table", c_ll)]


class _Rows(ctypes.Structure):
    """jc_kv_rows"""

    _fields_ = [("data", c_vp), ("ld", c_ll), ("head_stride", c_ll)]


_pc, _ps, _pr = ctypes.POINTER(_Cache), ctypes.POINTER(_Step), ctypes.POINTER(_Rows)
_lib.declare("jc_kv_append_device", c_int, [c_int, c_int, _pc, _ps, _pr, _pr, _pr, c_int, _pr, c_vp, c_vp, c_int, c_int,
                                            c_vp])
_lib.declare("jc_kv_attention_workspace", c_int, [c_int, _pc, _ps, c_int, c_int, c_int, ctypes.POINTER(c_ll)])
_lib.declare("jc_kv_attention_device", c_int, [c_int, c_int, _pc, _ps, _pr, c_int, _pr, c_int, c_int, ctypes.c_float,
                                               c_vp, c_ll, c_vp])
_lib.declare("jc_kv_read_device", c_int, [c_int, c_int, _pc, _ps, _pr, _pr, c_vp])


def rope_table(positions: int, head_dim: int, pairs: int | None = None, theta: float = 10000.0, device="cuda"):
    """The rotation table [positions, head_dim] (FP32: cosines of the head_dim / 2 pairs, then their sines) of
    ``pairs`` rotating pairs (default: all) of frequencies theta^(-e / pairs), as the engines build theirs: angles
    from FP32 position x FP32 frequency."""
    import numpy as np
    import torch

    pairs = head_dim // 2 if pairs is None else pairs
    exponent = (np.float32(2) * np.arange(pairs, dtype=np.float32)) / np.float32(2 * pairs)
    freq = np.float32(1) / np.power(np.float64(np.float32(theta)), exponent.astype(np.float64)).astype(np.float32)
    angle = (np.arange(positions, dtype=np.float32)[:, None] * freq).astype(np.float64)
    table = np.zeros((positions, head_dim), np.float32)
    table[:, :head_dim // 2] = 1.0  # pairs past the rotating ones stay
    table[:, :pairs] = np.cos(angle)
    table[:, head_dim // 2:head_dim // 2 + pairs] = np.sin(angle)
    return torch.from_numpy(table).to(device)


def _int32(t, name, dim, device=None):
    import torch

    if not torch.is_tensor(t) or t.dtype != torch.int32 or not t.is_cuda or t.dim() != dim or (
            dim and t.numel() and t.stride(-1) != 1):
        raise ValueError(f"{name} must be a {dim}-D int32 CUDA tensor with unit stride in its last dimension")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, not on {device}")
    return t


class Step:
    """The sequences of a call, shared by a model's layers: each one's cached ``length`` [n] (new tokens included)
    and its pages ``page_table`` [n, most pages], int32 on the GPU. ``start`` [n + 1] has the bounds of each
    sequence's packed new tokens (rows outside them are nobody's, their outputs are not written); without it every
    sequence has one. ``max_length`` and ``max_new`` bound the
    lengths and the new tokens, and may be set anew as series grow. The tensors stay those of the start; what they hold
    may be rewritten between calls (they are read on the GPU)."""

    length = property(lambda self: self._length)
    page_table = property(lambda self: self._page_table)
    start = property(lambda self: self._start)

    def __init__(self, length, page_table, max_length: int, start=None, max_new: int = 1):
        self._length = _int32(length, "length", 1)
        self.device = length.device
        self._page_table = _int32(page_table, "page_table", 2, self.device)
        n = length.shape[0]
        if page_table.shape[0] != n:
            raise ValueError(f"page_table has {page_table.shape[0]} rows for {n} sequences")
        if start is not None:
            _int32(start, "start", 1, self.device)
            if start.shape[0] != n + 1:
                raise ValueError(f"start has {start.shape[0]} bounds for {n} sequences")
        self._start, self.sequences = start, n
        self.max_length, self.max_new = max_length, max_new

    @property
    def max_length(self) -> int:
        return self._max_length

    @max_length.setter
    def max_length(self, value: int) -> None:
        if value < 0:
            raise ValueError("max_length must be >= 0")
        self._max_length = int(value)
        self._by_tokens = {}

    @property
    def max_new(self) -> int:
        return self._max_new

    @max_new.setter
    def max_new(self, value: int) -> None:
        if self._start is None and value != 1:
            raise ValueError("a step without start has one new token per sequence")
        if value < 0:
            raise ValueError("max_new must be >= 0")
        self._max_new = int(value)
        self._by_tokens = {}

    def _c(self, tokens: int):
        """The jc_kv_step over `tokens` packed rows."""
        got = self._by_tokens.get(tokens)
        if got is None:
            if self.start is None and tokens != self.sequences:
                raise ValueError(f"{tokens} rows for {self.sequences} sequences of one new token")
            ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
            got = ctypes.byref(_Step(self.sequences, tokens, self.max_new, self.max_length, ptr(self.start),
                                     ptr(self.length), ptr(self.page_table), self.page_table.shape[1],
                                     self.page_table.stride(0) if self.sequences > 1 else self.page_table.shape[1]))
            self._by_tokens = {tokens: got}
        return got


class PagedCache:
    """One layer's keys and values in pages of ``page_size`` tokens. ``k`` and ``v`` are the pools
    [pages, kv_heads, page_size, head_dim] (``bits`` 16) or their codes [.., head_dim // 2] with
    ``k_scale`` and ``v_scale`` [.., head_dim // 32, 2] (``bits`` 4), the same tensors for as long as it lives."""

    k = property(lambda self: self._pools[0])
    v = property(lambda self: self._pools[1])
    k_scale = property(lambda self: self._pools[2])
    v_scale = property(lambda self: self._pools[3])

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype=None, bits: int = 16,
                 device="cuda"):
        import torch

        shape = (pages, kv_heads, page_size)
        if bits == 16:
            dtype = torch.bfloat16 if dtype is None else dtype
            pool = lambda: torch.zeros((*shape, head_dim), dtype=dtype, device=device)  # noqa: E731
            self._bind(pool(), pool(), None, None)
        elif bits == 4:
            if dtype is not None:
                raise ValueError("a 4-bit cache has no dtype: its calls take theirs from their tensors")
            if head_dim % GROUP:
                raise ValueError(f"head_dim must be a multiple of {GROUP}")
            pool = lambda: torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device)  # noqa: E731
            scale = lambda: torch.zeros((*shape, head_dim // GROUP, 2), dtype=torch.float16, device=device)  # noqa: E731
            self._bind(pool(), pool(), scale(), scale())
        else:
            raise ValueError("bits must be 16 or 4")

    @classmethod
    def over(cls, k, v, k_scale=None, v_scale=None) -> "PagedCache":
        """A cache over pools that the caller holds."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale)
        return self

    def _bind(self, k, v, k_scale, v_scale) -> None:
        import torch

        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
            raise ValueError("k and v must be pools [pages, kv_heads, page_size, ..] of one shape and type")
        if k.dtype in (torch.bfloat16, torch.float16):
            if k_scale is not None or v_scale is not None:
                raise ValueError("a 16-bit cache has no scales")
            self.bits, dim = 16, k.shape[3]
        elif k.dtype == torch.uint8:
            self.bits, dim = 4, 2 * k.shape[3]
            for t in (k_scale, v_scale):
                if t is None or t.dtype != torch.float16 or tuple(t.shape) != (*k.shape[:3], dim // GROUP, 2):
                    raise ValueError(f"a 4-bit cache needs fp16 scales {(*k.shape[:3], dim // GROUP, 2)}")
        else:
            raise ValueError("pools must be bfloat16, float16, or uint8 (4-bit codes)")
        for t in (k, v, k_scale, v_scale):
            if t is not None and (not t.is_cuda or t.device != k.device or not t.is_contiguous()):
                raise ValueError("pools and scales must be contiguous CUDA tensors on one device")
        self._pools = (k, v, k_scale, v_scale)
        self.pages, self.kv_heads, self.page_size, self.head_dim = *k.shape[:3], dim
        self.device = k.device
        self.dtype = k.dtype if self.bits == 16 else None
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        self._c = ctypes.byref(_Cache(self.bits, self.pages, self.page_size, self.kv_heads, dim, ptr(k), ptr(v),
                                      ptr(k_scale), ptr(v_scale)))
        self._need = {}  # workspace bytes by the arguments that they depend on

    def _rows(self, t, name, heads=None, tokens=None, dtype=None):
        """jc_kv_rows of t [tokens, heads, head_dim]."""
        shape = t.shape
        if len(shape) != 3 or shape[2] != self.head_dim or t.device != self.device:
            raise ValueError(f"{name} must be [tokens, heads, {self.head_dim}] on {self.device}, not {tuple(shape)} on {t.device}")
        ld, hs, one = t.stride()
        if one != 1:
            raise ValueError(f"{name} must have unit stride in its last dimension")
        if heads is not None and shape[1] != heads:
            raise ValueError(f"{name} has {shape[1]} heads, not {heads}")
        if tokens is not None and shape[0] != tokens:
            raise ValueError(f"{name} has {shape[0]} tokens, not {tokens}")
        if dtype is not None and t.dtype != dtype:
            raise ValueError(f"{name} is {t.dtype}, not {dtype}")
        return ctypes.byref(_Rows(t.data_ptr(), ld, hs))

    def _precision(self, t) -> int:
        import torch

        if self.dtype is not None and t.dtype != self.dtype:
            raise ValueError(f"{t.dtype} tensors on a {self.dtype} cache")
        if t.dtype == torch.bfloat16:
            return BF16
        if t.dtype == torch.float16:
            return FP16
        raise ValueError(f"tensors must be bfloat16 or float16, not {t.dtype}")

    def _check_step(self, step: Step) -> None:
        if step.device != self.device:
            raise ValueError(f"the step is on {step.device}, the cache on {self.device}")

    def _stream(self) -> int:
        """torch's current stream on the cache's device (by the handle alone where torch offers it: a Stream object takes
        2 us, a fifth of a small call)."""
        import torch

        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        return raw(self.device.index) if raw else torch.cuda.current_stream(self.device).cuda_stream

    def append(self, step: Step, k, v, q=None, rope=None, pairs: int | None = None, positions=None, q_out=None):
        """Stores the step's new keys and values ``k``, ``v`` [tokens, kv_heads, head_dim]. With ``rope`` (a table,
        see ``rope_table``) keys and ``q`` [tokens, heads, head_dim] rotate in their first ``pairs`` pairs (default:
        all) by their index, or by ``positions`` [tokens] int32. Returns the rotated q (``q_out``, which may be q
        itself, or a new tensor), or None without q."""
        import torch

        self._check_step(step)
        n, dt = k.shape[0], k.dtype
        p = self._precision(k)
        rk = self._rows(k, "k", self.kv_heads)
        rv = self._rows(v, "v", self.kv_heads, n, dt)
        rq = ro = None
        heads = 0
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            rq = self._rows(q, "q", None, n, dt)
            if q_out is None:
                q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
                ro = ctypes.byref(_Rows(q_out.data_ptr(), heads * self.head_dim, self.head_dim))
            else:
                ro = self._rows(q_out, "q_out", heads, n, dt)
        elif q_out is not None:
            raise ValueError("q_out without q")
        rows, table = 0, None
        if rope is not None:
            if rope.dtype != torch.float32 or rope.dim() != 2 or rope.shape[1] != self.head_dim or (
                    not rope.is_contiguous()) or rope.device != self.device:
                raise ValueError(f"rope must be a contiguous fp32 table [positions, {self.head_dim}] on {self.device}")
            rows, table = rope.shape[0], rope.data_ptr()
            pairs = self.head_dim // 2 if pairs is None else pairs
        if positions is not None:
            _int32(positions, "positions", 1, self.device)
            if positions.shape[0] != n:
                raise ValueError(f"positions has {positions.shape[0]} entries for {n} tokens")
            positions = positions.data_ptr()
        check(_lib.lib().jc_kv_append_device(self.device.index, p, self._c, step._c(n), rk, rv, rq, heads, ro, positions,
                                             table, rows, pairs or 0, self._stream()))
        return q_out

    def attention(self, step: Step, q, window: int = 0, sinks: int = 0, scale: float | None = None, out=None):
        """Attention of the step's new tokens ``q`` [tokens, heads, head_dim] over the cache, which holds their keys
        already: each sees the keys up to its own, within ``window`` of it (0: all) or among the sequence's first
        ``sinks``. ``scale`` defaults to head_dim ** -0.5. Returns ``out`` (q itself, or a tensor beside it; a new one by
        default)."""
        import torch

        self._check_step(step)
        p = self._precision(q)
        rq = self._rows(q, "q")
        n, heads, dim = q.shape
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            ro = ctypes.byref(_Rows(out.data_ptr(), heads * dim, dim))
        else:
            ro = self._rows(out, "out", heads, n, q.dtype)
        c_step = step._c(n)
        lib = _lib.lib()
        key = (n, heads, window, sinks, step.sequences, step.max_new, step.max_length, p)
        need = self._need.get(key)
        if need is None:
            got = c_ll()
            check(lib.jc_kv_attention_workspace(p, self._c, c_step, heads, window, sinks, ctypes.byref(got)))
            if len(self._need) >= 64:
                self._need.clear()
            need = self._need[key] = got.value
        # from torch's allocator: the memory belongs to the current stream until its work is done
        work = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        check(lib.jc_kv_attention_device(self.device.index, p, self._c, c_step, rq, heads, ro, window, sinks,
                                         1.0 / math.sqrt(dim) if scale is None else scale,
                                         None if work is None else work.data_ptr(), need, self._stream()))
        return out

    def read(self, step: Step, tokens: int):
        """(k, v) [tokens, kv_heads, head_dim] of the step's new tokens from the cache (a step of n = length reads
        whole sequences): the cache's own values, or FP16 ones of a 4-bit cache. ``tokens``: the packed rows."""
        import torch

        self._check_step(step)
        k, v = (torch.empty((tokens, self.kv_heads, self.head_dim), dtype=self.dtype or torch.float16, device=self.device)
                for _ in range(2))
        check(_lib.lib().jc_kv_read_device(self.device.index, self._precision(k), self._c, step._c(tokens),
                                           self._rows(k, "k"), self._rows(v, "v"), self._stream()))
        return k, v
