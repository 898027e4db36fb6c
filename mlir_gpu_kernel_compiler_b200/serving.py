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
which skips it and records it: ``check()`` raises for it.  Indices are int32; int64 ones are narrowed by a launch
of their own.

Gradients: ``rotary`` has one, its inverse, and so has the turned ``q`` of ``rotary_cache_write``.  Attention has none:
its result raises in the backward pass.  A cache keeps values, not what they came from, so nothing flows back
through it.

Each operator is a C entry point of ``include/tj_b200.h`` over hand-written sm_100a kernels in
``csrc/serving``.
"""
from __future__ import annotations

import ctypes
import importlib.util
import math
from typing import Optional

import torch

from . import runtime as rt
from . import toolchain

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8,
          "e4m3": torch.float8_e4m3fn}


def _load():
    """The binding (``csrc/serving/serving_module.cpp``), built in-tree first if it is missing."""
    spec = importlib.util.spec_from_file_location("_serving", toolchain.build_serving_module())
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    rt.library()
    module.init(str(toolchain.build_runtime()), rt.RuntimeError_, torch.OutOfMemoryError)
    return module


_native = _load()


class PagedCache:
    """A pool of pages of keys and values; borrows its tensors, which cannot be replaced.

    ``k`` and ``v``: ``[pages, page_size, kv_heads, head_dim]``, f16 or bf16, or i8 or e4m3 codes with
    scales ``[pages, page_size, kv_heads]`` in f32 (value = code * scale).  Both may be views whose
    memory is in another order (heads before slots, say), the same for k and v, rows contiguous and
    starting on 16-byte boundaries (8-byte ones do for 8-bit codes that attention does not read).
    Slot ``s`` is place ``s % page_size`` of page ``s // page_size``.
    """

    __slots__ = ("_tensors", "_native")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        self._native = _native.describe(k, v, k_scale, v_scale)
        self._tensors = k, v, k_scale, v_scale

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    device = property(lambda self: self.k.device)
    dtype = property(lambda self: self.k.dtype)
    pages = property(lambda self: self.k.shape[0])
    page_size = property(lambda self: self.k.shape[1])
    kv_heads = property(lambda self: self.k.shape[2])
    head_dim = property(lambda self: self.k.shape[3])

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


def _described(cache) -> bytes:
    if type(cache) is not PagedCache:
        raise TypeError(f"cache: expected a PagedCache, got {type(cache).__name__}")
    return cache._native


class _Rotary(torch.autograd.Function):
    """Turning is linear, and turning back is its transpose (whatever the table's magnitude)."""

    @staticmethod
    def forward(ctx, q, k, positions, table, layout, inverse):
        ctx.save_for_backward(positions, table)
        ctx.how = layout, inverse, k is None
        return _native.rotary(q, k, positions, table, layout, inverse, None)

    @staticmethod
    def backward(ctx, q_grad, k_grad):
        layout, inverse, alone = ctx.how
        q_grad, k_grad = rotary(q_grad, None if alone else k_grad, *ctx.saved_tensors, layout=layout, inverse=not inverse)
        return q_grad, k_grad, None, None, None, None


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, *args):
        return _native.attention(args[0], q, *args[1:])

    @staticmethod
    def backward(ctx, *grads):
        raise NotImplementedError("paged_attention has no gradient: call it under torch.no_grad()")


def rotary(q, k, positions, table, *, layout: str = "half", inverse: bool = False, out=None):
    """Rotary positions on ``q`` and ``k`` (``k`` may be None): ``(q', k')``.

    ``[tokens, heads, head_dim]`` in f32, f16 or bf16, head_dim a multiple of 8 up to 512; the first
    ``table.shape[1]`` elements of a row are turned, the rest passed on.  ``layout``: pairs
    ``(i, i + rot / 2)`` ("half") or ``(2 i, 2 i + 1)`` ("interleaved").  ``inverse`` turns by the opposite angles, which
    undoes the turn (times the square of a table's magnitude) and is also the gradient's pass; autograd follows
    the call.  ``out``: ``(q', k')`` to write, which may be q and k themselves (not under autograd).
    """
    got = _native.rotary(q, k, positions, table, layout, inverse, out)
    return _Rotary.apply(q, k, positions, table, layout, inverse) if got is NotImplemented else got


def cache_write(cache: PagedCache, k, v, slots) -> None:
    """Tokens' keys and values ``[tokens, kv_heads, head_dim]`` (f32, f16 or bf16) into the cache's slots.

    An i8 or e4m3 cache gets, for each (token, head), ``scale = max|x| / 127`` (``/ 448``) and the codes
    of ``x / scale``, rounded to nearest even; a row with an infinity or a NaN is held as NaN.  A negative
    slot skips its token; two tokens must not share a slot.
    """
    _native.write(_described(cache), None, k, v, slots, None, None, "half", None)


def rotary_cache_write(cache: PagedCache, q, k, v, slots, positions, table, *, layout: str = "half", out=None):
    """``rotary`` on ``q`` and ``k`` and ``cache_write`` of the turned keys and of ``v``, in one launch: ``q'``.

    The keys go from f32 into the cache's type without a rounding between.  ``q`` may be None.
    """
    if table is None or positions is None:
        raise TypeError("rotary_cache_write needs positions and a table")
    got = _native.write(_described(cache), q, k, v, slots, positions, table, layout, out)
    if got is NotImplemented:  # q's turn goes into autograd's graph
        _native.write(_described(cache), None, k, v, slots, positions, table, layout, None)
        got = rotary(q, None, positions, table, layout=layout)[0]
    return got


def cache_read(cache: PagedCache, slots, dtype: str = "bf16") -> tuple[torch.Tensor, torch.Tensor]:
    """Slots' keys and values as dense rows ``[len(slots), kv_heads, head_dim]``; a negative slot reads as 0."""
    return _native.read(_described(cache), slots, dtype)


def paged_attention(q, cache: PagedCache, page_table, kv_lens, q_starts=None, *, max_new: Optional[int] = None,
                    scale: Optional[float] = None, causal: bool = True, window: int = 0, return_lse: bool = False, out=None):
    """Attention of new tokens over their sequences' cached keys and values: ``[tokens, q_heads, head_dim]``.

    ``q``: f16 or bf16, head_dim 64 or 128, q_heads a multiple of the cache's heads (query heads
    ``h * group .. (h + 1) * group`` read cached head ``h``).  A 16-bit cache has q's dtype.
    ``page_table`` int32 ``[batch, width]``: the pages of each sequence in order; ``kv_lens`` ``[batch]``: its
    keys, the new tokens' among them (written before the call); ``q_starts`` ``[batch + 1]``: its new
    tokens are rows ``q_starts[b]`` to ``q_starts[b + 1]`` of q, the last of its keys (None: one each); it
    does not descend.
    ``max_new``: the most new tokens of any sequence (default: 1 without q_starts, else not known).  It helps to
    choose the kernel and nothing else; with it, rows of no sequence change no bit of the others.

    A token sees the keys up to its own position; if not ``causal``, those after it too.  A positive ``window``
    hides the keys before the last ``window`` up to its own position (its own among them), and, without the
    causal mask, none of those after it.  ``scale`` (default head_dim**-0.5) multiplies the scores.  A row that
    sees no key is 0; rows of no sequence are not written.  ``return_lse``: also the logarithm of each row's sum
    of exponentials, f32 ``[tokens, q_heads]`` (-inf for a row that sees no key).  Slots that no row of a
    sequence sees may hold anything; visible ones must be finite, as a NaN or an infinity reaches the
    sequence's other rows too.  Value scales of an 8-bit cache up to 2**20 (values of 1e8) are exact to f32 beside any
    others; beside larger ones the weights of keys with much smaller values may be lost.

    A call needs a workspace (a partial result of 16 or 256 rows for each CTA, some MB to some hundred for thousands of
    sequences), which is kept for each stream.
    """
    how = page_table, kv_lens, q_starts, max_new, scale, causal, window, return_lse, out
    got = _native.attention(_described(cache), q, *how)
    return _Attention.apply(q, _described(cache), *how) if got is NotImplemented else got


_OPERATORS = ("rotary", "cache_write", "cache_read", "paged_attention")
_SITES = {1: "slot", 2: "position", 3: "page", 4: "length", 6: "q_starts"}


def check(device="cuda") -> None:
    """Synchronise the current stream and raise if a serving operator met an index out of range since the
    last check (its row or token was skipped; turned by a position out of range, a row became NaN; with
    ``q_starts`` in descending order attention did nothing), or a bounded wait of a kernel ran out."""
    device = torch.device(device)
    if device.index is None:
        device = torch.device(device.type, torch.cuda.current_device())
    code, where = ctypes.c_int32(), ctypes.c_int32()
    with torch.cuda.device(device):
        rc = rt.library().tj_b200_serving_status(ctypes.byref(code), ctypes.byref(where), torch.cuda.current_stream(device).cuda_stream)
    if rc == rt.TJ_ERR_DEVICE_STATUS:
        if code.value == 1:
            _native.forget()  # a kernel that gave up may have left its counters as they were
        op, site = _OPERATORS[where.value // 16 % 4], where.value % 16
        what = f"{_SITES[site]} out of range" if code.value == 2 else f"wait timeout (site {site})"
        raise rt.RuntimeError_(rc, f"{op}: {what}")
    rt.check(rc, "tj_b200_serving_status")
