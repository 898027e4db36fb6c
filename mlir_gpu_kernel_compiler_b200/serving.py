"""Serving operators: rotary positions, a paged cache of keys and values, attention over it.

A compiled program (``B200Program``) maps inputs to outputs and keeps nothing between calls.  A
decoder keeps the keys and values of the tokens that it has seen; these operators are that part,
called between the programs of a layer:

    table = serving.rotary_table(128, 32768, device="cuda")
    cache = serving.PagedCache.empty(pages=4096, page_size=16, kv_heads=8, head_dim=128, dtype="i8")
    q = serving.rotary_cache_write(cache, q, k, v, slots, positions, table)     # new tokens
    o = serving.paged_attention(q, cache, page_table, kv_lens, q_starts, max_new=64)

Tensors are ``[tokens, heads, head_dim]``; any strides whose rows are contiguous are read in place
(the three slices of a fused projection, say).  Calls run on torch's current stream of the
tensors' device and return without waiting.  As in ``B200Program``, a wrong type raises
``TypeError``, a wrong shape, dtype or device ``ValueError``, a failed launch
``runtime.RuntimeError_``; a slot, position, page or length out of range is seen by the device alone,
which skips it and records it: ``check()`` raises for it.

Each operator is one hand-written sm_100a kernel in ``csrc/serving`` behind a C entry point of
``include/tj_b200.h``.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch

from . import runtime as rt

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
          "e4m3": torch.float8_e4m3fn}
_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_ROWS = (torch.float32, torch.float16, torch.bfloat16)
_UNIT = {torch.float32: 4, torch.float16: 8, torch.bfloat16: 8}  # elements in 16 bytes

_CACHE = struct.Struct("=15q")            # tj_kv_cache
_TJ_ROWS = struct.Struct("=27q")          # tj_rows, without its cache
_ATTENTION = struct.Struct("=21qd2q")     # tj_paged_attention, without its cache


def _expect(t, name: str, dim: int, dtypes, device=None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.dim() != dim:
        raise ValueError(f"{name}: expected {dim} dimensions, got shape {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype} is not supported (one of {', '.join(map(str, dtypes))})")
    if t.device.type != "cuda" or (device is not None and t.device != device):
        raise ValueError(f"{name}: tensor is on {t.device}, not on {device or 'a CUDA device'}")


def _indices(t, name: str, device, size: int) -> torch.Tensor:
    """A vector of ``size`` 32-bit indices, contiguous."""
    _expect(t, name, 1, (torch.int32, torch.int64), device)
    if t.shape[0] != size:
        raise ValueError(f"{name}: expected {size} entries, got {t.shape[0]}")
    return t if t.dtype is torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """Rows the kernels can read with 16-byte loads: the tensor itself, or a copy."""
    st, sh, sd = t.stride()
    unit = _UNIT[t.dtype]
    if sd == 1 and not (st % unit or sh % unit or t.data_ptr() % 16):
        return t
    return t.contiguous() if t.data_ptr() % 16 == 0 and not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)


def _out_rows(out, name: str, like: torch.Tensor) -> torch.Tensor:
    _expect(out, name, 3, (like.dtype,), like.device)
    if out.shape != like.shape:
        raise ValueError(f"{name}: expected shape {tuple(like.shape)}, got {tuple(out.shape)}")
    st, sh, sd = out.stride()
    unit = _UNIT[out.dtype]
    if (sd != 1 or st % unit or sh % unit or out.data_ptr() % 16) and out.numel():
        raise ValueError(f"{name}: rows must be contiguous and start on 16-byte boundaries")
    return out


class _on:
    """The device of a call, made current for the launch if it is not; its current stream."""

    __slots__ = ("index", "old", "stream")

    def __init__(self, device: torch.device):
        self.index = device.index

    def __enter__(self):
        self.old = torch.cuda.current_device()
        if self.old != self.index:
            torch.cuda.set_device(self.index)
        self.stream = torch._C._cuda_getCurrentRawStream(self.index)
        return self

    def __exit__(self, *exc):
        if self.old != self.index:
            torch.cuda.set_device(self.old)


class PagedCache:
    """A pool of pages of keys and values; borrows its tensors.

    ``k`` and ``v``: ``[pages, page_size, kv_heads, head_dim]``, f16 or bf16, or i8 or e4m3 codes with
    scales ``[pages, page_size, kv_heads]`` in f32 (value = code * scale).  Both may be views whose
    memory is in another order (heads before slots, say), the same for k and v, rows contiguous.
    Slot ``s`` is place ``s % page_size`` of page ``s // page_size``.
    """

    __slots__ = ("k", "v", "k_scale", "v_scale", "packed", "device", "dtype", "pages", "page_size", "kv_heads", "head_dim")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        _expect(k, "k", 4, tuple(_CODE)[1:])
        _expect(v, "v", 4, (k.dtype,), k.device)
        shape, strides = k.shape, k.stride()
        if v.shape != shape or v.stride() != strides:
            raise ValueError("k and v must have the same shape and strides")
        size = k.element_size()
        pages, page_size, heads, dim = shape
        if dim % 8 or not 0 < dim <= 512:
            raise ValueError(f"head dim {dim} is not a multiple of 8 from 8 to 512")
        unit = 8 if size == 1 else 16
        if strides[3] != 1 or any(s * size % unit for s in strides[:3]) or (k.data_ptr() | v.data_ptr()) % 16:
            raise ValueError(f"cache rows must be contiguous and start on {unit}-byte boundaries")
        scale_at = (0, 0, 0)
        if size == 1:
            for t, name in ((k_scale, "k_scale"), (v_scale, "v_scale")):
                if t is None:
                    raise ValueError(f"a {k.dtype} cache needs {name}")
                _expect(t, name, 3, (torch.float32,), k.device)
                if t.shape != shape[:3]:
                    raise ValueError(f"{name}: expected shape {tuple(shape[:3])}, got {tuple(t.shape)}")
            scale_at = k_scale.stride()
            if v_scale.stride() != scale_at:
                raise ValueError("k_scale and v_scale must have the same strides")
        elif k_scale is not None or v_scale is not None:
            raise ValueError(f"a {k.dtype} cache has no scales")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.device, self.dtype = k.device, k.dtype
        self.pages, self.page_size, self.kv_heads, self.head_dim = pages, page_size, heads, dim
        self.packed = _CACHE.pack(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if size == 1 else 0,
                                  v_scale.data_ptr() if size == 1 else 0, pages, page_size, heads, dim, *strides[:3],
                                  *scale_at, _CODE[k.dtype])

    @classmethod
    def empty(cls, pages: int, page_size: int, kv_heads: int, head_dim: int, dtype: str = "bf16", device="cuda",
              heads_first: bool = False) -> "PagedCache":
        """A zeroed cache.  ``heads_first``: a page's memory is [kv_heads, page_size, head_dim]."""
        if dtype not in ("f16", "bf16", "i8", "e4m3"):
            raise ValueError(f"dtype must be f16, bf16, i8 or e4m3, not {dtype!r}")

        def pool():
            if heads_first:
                return torch.zeros(pages, kv_heads, page_size, head_dim, dtype=DTYPES[dtype], device=device).transpose(1, 2)
            return torch.zeros(pages, page_size, kv_heads, head_dim, dtype=DTYPES[dtype], device=device)

        scales = [None, None]
        if dtype in ("i8", "e4m3"):
            scales = [torch.zeros(pages, page_size, kv_heads, device=device) for _ in range(2)]
        return cls(pool(), pool(), *scales)


def rotary_table(rot_dim: int, max_positions: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                 original: int = 0, fast: float = 32.0, slow: float = 1.0, magnitude: float = 1.0, device="cuda") -> torch.Tensor:
    """cos and sin of the rotary angles: f32 ``[max_positions, rot_dim]``, cosines then sines.

    Pair ``i`` turns by ``position * base**(-2 i / rot_dim)``, computed in 64 bits.  For contexts
    ``factor`` times longer than a model was trained on, ``scaling`` is one of

    * ``"linear"``: every frequency divided by ``factor``;
    * ``"base"``: ``base`` times ``factor**(rot_dim / (rot_dim - 2))``, so that the slowest pair slows
      down by ``factor`` and the fastest keeps its frequency;
    * ``"ramp"``: pairs that turn at least ``fast`` times within ``original`` positions keep their
      frequency, those that turn at most ``slow`` times are divided by ``factor``, with a linear ramp in
      the number of turns between.

    ``magnitude`` multiplies every entry (it scales the scores by its square).
    """
    if rot_dim <= 0 or rot_dim % 2 or max_positions <= 0:
        raise ValueError("rot_dim must be even and positive, max_positions positive")
    if scaling not in (None, "linear", "base", "ramp"):
        raise ValueError(f"scaling must be None, 'linear', 'base' or 'ramp', not {scaling!r}")
    if factor <= 0 or (scaling == "base" and rot_dim < 4) or (scaling == "ramp" and (original <= 0 or not fast > slow)):
        raise ValueError("factor must be positive; 'base' needs rot_dim >= 4; 'ramp' needs original > 0 and fast > slow")
    half = rot_dim // 2
    if scaling == "base":
        base = base * factor ** (rot_dim / (rot_dim - 2))
    freq = base ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "ramp":
        keep = ((original * freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return (torch.cat((angle.cos(), angle.sin()), 1) * magnitude).float()


def _check_table(table, positions, device, tokens: int, dim: int, layout: str):
    _expect(table, "table", 2, (torch.float32,), device)
    if layout not in ("half", "interleaved"):
        raise ValueError(f"layout must be 'half' or 'interleaved', not {layout!r}")
    rot = table.shape[1]
    if rot % 2 or not 0 < rot <= dim or table.shape[0] == 0:
        raise ValueError(f"table: {rot} columns do not turn rows of {dim}")
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    return table, _indices(positions, "positions", device, tokens)


_NO_CACHE = bytes(_CACHE.size)


def rotary(q, k, positions, table, *, layout: str = "half", inverse: bool = False, out=None):
    """Rotary positions on ``q`` and ``k`` (``k`` may be None): ``(q', k')``.

    ``[tokens, heads, head_dim]`` in f32, f16 or bf16, head_dim a multiple of 8 up to 512; the first
    ``table.shape[1]`` elements of a row are turned, the rest passed on.  ``layout``: pairs
    ``(i, i + rot / 2)`` ("half") or ``(2 i, 2 i + 1)`` ("interleaved").  ``inverse`` turns back, which is
    also the gradient's pass.  ``out``: ``(q', k')`` to write, which may be q and k themselves.
    """
    _expect(q, "q", 3, _ROWS)
    tokens, heads, dim = q.shape
    if dim % 8 or not 0 < dim <= 512:
        raise ValueError(f"head dim {dim} is not a multiple of 8 from 8 to 512")
    table, positions = _check_table(table, positions, q.device, tokens, dim, layout)
    if k is not None:
        _expect(k, "k", 3, (q.dtype,), q.device)
        if k.shape[0] != tokens or k.shape[2] != dim:
            raise ValueError(f"k: shape {tuple(k.shape)} does not go with q's {tuple(q.shape)}")
    if out is None:
        q2 = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
        k2 = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    else:
        q2 = _out_rows(out[0], "out[0]", q)
        k2 = None if k is None else _out_rows(out[1], "out[1]", k)
    q, k = _rows(q), None if k is None else _rows(k)
    ks = (0, 0) if k is None else k.stride()
    k2s = (0, 0) if k is None else k2.stride()
    qs, q2s = q.stride(), q2.stride()
    args = _TJ_ROWS.pack(
        q.data_ptr(), 0 if k is None else k.data_ptr(), 0, q2.data_ptr(), 0 if k is None else k2.data_ptr(), 0,
        positions.data_ptr(), table.data_ptr(), tokens, heads, 0 if k is None else k.shape[1], dim, table.shape[1],
        table.shape[0], qs[0], qs[1], ks[0], ks[1], 0, 0, q2s[0], q2s[1], k2s[0], k2s[1], _CODE[q.dtype],
        layout == "interleaved", inverse)
    with _on(q.device) as on:
        rc = rt.library().tj_b200_rotary(args + _NO_CACHE, on.stream)
    if rc:
        rt.check(rc)
    return q2, k2


def _write(cache, q, k, v, slots, positions, table, layout, out):
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache: expected a PagedCache, got {type(cache).__name__}")
    device = cache.device
    _expect(k, "k", 3, _ROWS, device)
    _expect(v, "v", 3, (k.dtype,), device)
    tokens, heads, dim = k.shape
    if v.shape != k.shape or heads != cache.kv_heads or dim != cache.head_dim:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not go with a cache of {cache.kv_heads} heads of {cache.head_dim}")
    slots = _indices(slots, "slots", device, tokens)
    rot = rows = q_heads = q_ptr = q2_ptr = pos_ptr = table_ptr = 0
    q2, qs, q2s = None, (0, 0), (0, 0)
    if table is not None:
        table, positions = _check_table(table, positions, device, tokens, dim, layout)
        rot, rows, pos_ptr, table_ptr = table.shape[1], table.shape[0], positions.data_ptr(), table.data_ptr()
        if q is not None:
            _expect(q, "q", 3, (k.dtype,), device)
            if q.shape[0] != tokens or q.shape[2] != dim:
                raise ValueError(f"q: shape {tuple(q.shape)} does not go with k's {tuple(k.shape)}")
            q_heads = q.shape[1]
            q2 = torch.empty((tokens, q_heads, dim), dtype=q.dtype, device=device) if out is None else _out_rows(out, "out", q)
            q = _rows(q)
            q_ptr, q2_ptr, qs, q2s = q.data_ptr(), q2.data_ptr(), q.stride(), q2.stride()
    k, v = _rows(k), _rows(v)
    ks, vs = k.stride(), v.stride()
    args = _TJ_ROWS.pack(q_ptr, k.data_ptr(), v.data_ptr(), q2_ptr, 0, slots.data_ptr(), pos_ptr, table_ptr, tokens, q_heads,
                         heads, dim, rot, rows, qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], q2s[0], q2s[1], 0, 0, _CODE[k.dtype],
                         layout == "interleaved", 0)
    with _on(device) as on:
        rc = rt.library().tj_b200_cache_write(args + cache.packed, on.stream)
    if rc:
        rt.check(rc)
    return q2


def cache_write(cache: PagedCache, k, v, slots) -> None:
    """Tokens' keys and values ``[tokens, kv_heads, head_dim]`` (f32, f16 or bf16) into the cache's slots.

    An i8 or e4m3 cache gets, for each (token, head), ``scale = max|x| / 127`` (``/ 448``) and the codes
    of ``x / scale``, rounded to nearest even; a row with an infinity or a NaN is held as NaN.  A negative
    slot skips its token; two tokens must not share a slot.
    """
    _write(cache, None, k, v, slots, None, None, "half", None)


def rotary_cache_write(cache: PagedCache, q, k, v, slots, positions, table, *, layout: str = "half", out=None):
    """``rotary`` on ``q`` and ``k`` and ``cache_write`` of the turned keys and of ``v``, in one launch: ``q'``.

    The keys go from f32 into the cache's type without a rounding between.  ``q`` may be None.
    """
    if table is None or positions is None:
        raise TypeError("rotary_cache_write needs positions and a table")
    return _write(cache, q, k, v, slots, positions, table, layout, out)


def cache_read(cache: PagedCache, slots, dtype: str = "bf16") -> tuple[torch.Tensor, torch.Tensor]:
    """Slots' keys and values as dense rows ``[len(slots), kv_heads, head_dim]``; a negative slot reads as 0."""
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache: expected a PagedCache, got {type(cache).__name__}")
    if dtype not in ("f32", "f16", "bf16"):
        raise ValueError(f"dtype must be f32, f16 or bf16, not {dtype!r}")
    if not isinstance(slots, torch.Tensor):
        raise TypeError(f"slots: expected a torch.Tensor, got {type(slots).__name__}")
    n = slots.shape[0] if slots.dim() == 1 else -1
    slots = _indices(slots, "slots", cache.device, n)
    kind = DTYPES[dtype]
    k = torch.empty((n, cache.kv_heads, cache.head_dim), dtype=kind, device=cache.device)
    v = torch.empty_like(k)
    with _on(cache.device) as on:
        rc = rt.library().tj_b200_cache_read(cache.packed, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), _CODE[kind], on.stream)
    if rc:
        rt.check(rc)
    return k, v


# A call's workspace and its counters (zero between calls), kept for each stream: calls on one stream
# follow one another, calls on two must not share them.
_workspaces: dict[tuple, tuple[torch.Tensor, torch.Tensor]] = {}
_needs: dict[tuple, tuple[int, int]] = {}


def _workspace(device, stream: int, key: tuple, args: bytes):
    need = _needs.get(key)
    if need is None:
        size, count = ctypes.c_int64(), ctypes.c_int64()
        rt.check(rt.library().tj_b200_paged_attention_workspace(args, ctypes.byref(size), ctypes.byref(count)),
                 "tj_b200_paged_attention_workspace")
        if len(_needs) > 4096:
            _needs.clear()
        need = _needs[key] = (size.value, count.value)
    if torch.cuda.is_current_stream_capturing():
        # a graph's own: its zeroing is part of the graph, its memory belongs to the graph's pool
        return (torch.empty(need[0], dtype=torch.uint8, device=device),
                torch.zeros(need[1], dtype=torch.int32, device=device), need)
    held = _workspaces.get((device, stream))
    if held is None or held[0].shape[0] < need[0] or held[1].shape[0] < need[1]:
        size, count = (0, 0) if held is None else (held[0].shape[0], held[1].shape[0])
        held = (torch.empty(max(size, need[0]), dtype=torch.uint8, device=device),
                torch.zeros(max(count, need[1]), dtype=torch.int32, device=device))
        _workspaces[(device, stream)] = held
    return held[0], held[1], need


def paged_attention(q, cache: PagedCache, page_table, kv_lens, q_starts=None, *, max_new: Optional[int] = None,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0, return_lse: bool = False, out=None):
    """Attention of new tokens over their sequences' cached keys and values: ``[tokens, q_heads, head_dim]``.

    ``q``: f16 or bf16, head_dim 64 or 128, q_heads a multiple of the cache's heads (query heads
    ``h * group .. (h + 1) * group`` read cached head ``h``).  A 16-bit cache has q's dtype.
    ``page_table`` int32 ``[batch, width]``: the pages of each sequence in order; ``kv_lens`` ``[batch]``: its
    keys, the new tokens' among them (written before the call); ``q_starts`` ``[batch + 1]``: its new
    tokens are rows ``q_starts[b]`` to ``q_starts[b + 1]`` of q, the last of its keys (None: one each).
    ``max_new``: the most new tokens of any sequence (default: 1 without q_starts, else all of them).

    A token sees the keys up to its own position (all of them if not ``causal``), of those the last
    ``window`` if that is positive.  ``scale`` (default head_dim**-0.5) multiplies the scores.  A row that
    sees no key is 0; rows of no sequence are not written.  ``return_lse``: also the logarithm of each row's sum
    of exponentials, f32 ``[tokens, q_heads]`` (-inf for a row that sees no key).  Slots that no row of a
    sequence sees may hold anything; visible ones must be finite, as a NaN or an infinity reaches the
    sequence's other rows too.
    """
    if not isinstance(cache, PagedCache):
        raise TypeError(f"cache: expected a PagedCache, got {type(cache).__name__}")
    device, dim = cache.device, cache.head_dim
    _expect(q, "q", 3, (torch.float16, torch.bfloat16), device)
    tokens, heads, qdim = q.shape
    if qdim != dim or heads % cache.kv_heads or heads == 0:
        raise ValueError(f"q: shape {tuple(q.shape)} does not go with a cache of {cache.kv_heads} heads of {dim}")
    if dim not in (64, 128):
        raise ValueError(f"head dim must be 64 or 128, not {dim}")
    if cache.dtype in _ROWS and cache.dtype != q.dtype:
        raise ValueError(f"q is {q.dtype} and the cache {cache.dtype}: a 16-bit cache must have q's dtype")
    _expect(page_table, "page_table", 2, (torch.int32, torch.int64), device)
    if page_table.dtype is not torch.int32 or page_table.stride(1) != 1:
        page_table = page_table.to(torch.int32).contiguous()
    batch, width = page_table.shape
    if width == 0 and batch:
        raise ValueError("page_table: no columns")
    kv_lens = _indices(kv_lens, "kv_lens", device, batch)
    starts = 0
    if q_starts is not None:
        q_starts = _indices(q_starts, "q_starts", device, batch + 1)
        starts = q_starts.data_ptr()
    elif tokens != batch:
        raise ValueError(f"without q_starts there is one token to a sequence: {tokens} tokens, {batch} sequences")
    if max_new is None:
        max_new = 1 if q_starts is None else max(tokens, 1)
    if max_new < 1 or window < 0:
        raise ValueError("max_new must be positive and window not negative")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < math.inf:
        raise ValueError("scale must be positive")
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=device)
    else:
        out = _out_rows(out, "out", q)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    if tokens and batch:
        q = _rows(q)
        qs, os_ = q.stride(), out.stride()
        with _on(device) as on:
            key = (device, cache.dtype, dim, cache.kv_heads, heads, tokens, batch, max_new, starts != 0)
            fields = [q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, page_table.data_ptr(), kv_lens.data_ptr(),
                      starts, 0, 0, tokens, batch, heads, max_new, page_table.stride(0), width, qs[0], qs[1], os_[0], os_[1],
                      _CODE[q.dtype], causal, window, scale, 0, 0]
            workspace, counters, need = _workspace(device, on.stream, key, _ATTENTION.pack(*fields) + cache.packed)
            fields[6], fields[7], fields[22], fields[23] = workspace.data_ptr(), counters.data_ptr(), need[0], need[1]
            rc = rt.library().tj_b200_paged_attention(_ATTENTION.pack(*fields) + cache.packed, on.stream)
        if rc:
            rt.check(rc)
    return (out, lse) if return_lse else out


_OPERATORS = ("rotary", "cache_write", "cache_read", "paged_attention")
_SITES = {1: "slot", 2: "position", 3: "page", 4: "length"}


def check(device="cuda") -> None:
    """Synchronise the current stream and raise if a serving operator met an index out of range since the
    last check (its row or token was skipped), or a bounded wait of a kernel ran out."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    code, where = ctypes.c_int32(), ctypes.c_int32()
    with _on(device) as on:
        rc = rt.library().tj_b200_serving_status(ctypes.byref(code), ctypes.byref(where), on.stream)
    if rc == rt.TJ_ERR_DEVICE_STATUS:
        op, site = _OPERATORS[where.value // 16 % 4], where.value % 16
        what = f"{_SITES[site]} out of range" if site in _SITES else f"wait timeout (site {site})"
        raise rt.RuntimeError_(rc, f"{op}: {what}")
    rt.check(rc, "tj_b200_serving_status")
