"""The serving operators against plain implementations in 64 bits.

Tolerances, from the formats: u is the unit roundoff of a 16-bit type (2^-8 bf16, 2^-11 f16).  A rotated
element is two products and a sum in f32 and one rounding.  An attention output is one rounding of
itself and one of each probability, u (|o| + sum p |v|), plus the f32 error of the scores' exponent,
2e-5 sum p |v| for scores up to a few hundred.  Codes of a quantised cache follow from IEEE
operations in f32 and have to be equal.
"""
import math

import pytest
import torch

from mlir_gpu_kernel_compiler_b200 import runtime as rt
from mlir_gpu_kernel_compiler_b200 import serving

pytestmark = pytest.mark.gpu
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-23}
DT = serving.DTYPES
TOP = {"i8": 127.0, "e4m3": 448.0}


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    serving.check()


def _gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(*shape, dtype=torch.float32, seed=0, scale=1.0):
    return (torch.randn(*shape, device="cuda", generator=_gen(seed)) * scale).to(dtype)


# ---- rotary ------------------------------------------------------------------------------------


def _turn64(x, positions, table, layout, inverse=False):
    x, row = x.double(), table.double()[positions.long()]
    rot = table.shape[1]
    half = rot // 2
    unit = torch.complex(row[:, :half], row[:, half:] * (-1 if inverse else 1))[:, None]
    y = x.clone()
    if layout == "half":
        z = torch.complex(x[..., :half], x[..., half:rot]) * unit
        y[..., :half], y[..., half:rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * unit
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def _rot_tol(x, u):
    # |a| + |b| bounds both products; three f32 roundings of them and one to the type
    return u * 1.01 * x.double().abs() + 2.0**-22 * x.double().abs().amax(-1, keepdim=True) + 1e-30


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot", [(1, 1, 1, 8, 2), (1, 32, 8, 128, 128), (7, 5, 3, 80, 20), (33, 4, 4, 96, 96),
                                                  (301, 8, 1, 64, 32), (5, 3, 2, 512, 48), (3, 2, 2, 72, 72), (2, 7, 7, 256, 6)])
def test_rotary(layout, dtype, tokens, hq, hk, dim, rot):
    table = serving.rotary_table(rot, 4096)
    q, k = _randn(tokens, hq, dim, dtype=DT[dtype], seed=1), _randn(tokens, hk, dim, dtype=DT[dtype], seed=2)
    pos = torch.randint(0, 4096, (tokens,), device="cuda", generator=_gen(3))
    for inverse in (False, True):
        for x, y in zip((q, k), serving.rotary(q, k, pos, table, layout=layout, inverse=inverse)):
            want = _turn64(x, pos, table, layout, inverse)
            assert y.dtype == x.dtype
            assert ((y.double() - want).abs() <= _rot_tol(want, U[x.dtype])).all()
            assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [64, 20])
def test_rotary_strided_in_place_and_without_keys(layout, rot):
    table = serving.rotary_table(rot, 512)
    pos = torch.arange(40, device="cuda").int()
    rows = _randn(40, 7, 64, dtype=torch.bfloat16)
    want_q, want_k = serving.rotary(rows[:, :4].clone(), rows[:, 4:6].clone(), pos, table, layout=layout)
    got_q, got_k = serving.rotary(rows[:, :4], rows[:, 4:6], pos, table, layout=layout)
    assert torch.equal(got_q, want_q) and torch.equal(got_k, want_k)
    odd = torch.zeros(40, 4, 67, device="cuda", dtype=torch.bfloat16)[..., 3:]  # rows at odd addresses
    odd.copy_(rows[:, :4])
    alone, none = serving.rotary(odd, None, pos, table, layout=layout)
    assert none is None and torch.equal(alone, want_q)
    last = rows[:, 6].clone()
    serving.rotary(rows[:, :4], rows[:, 4:6], pos, table, layout=layout, out=(rows[:, :4], rows[:, 4:6]))
    assert torch.equal(rows[:, :4], want_q) and torch.equal(rows[:, 4:6], want_k) and torch.equal(rows[:, 6], last)
    by_head = want_q.transpose(0, 1).contiguous().transpose(0, 1)
    back, _ = serving.rotary(by_head, None, pos, table, layout=layout, inverse=True)
    assert ((back.double() - odd.double()).abs() <= 3 * 2.0**-8 * odd.double().abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_gradient(layout):
    """d/dx <w, rotary(x)> is rotary(w, inverse): against 64-bit autograd and against differences (the map is
    linear, so a difference over any step is exact up to the rounding of f32)."""
    table = serving.rotary_table(24, 64)
    pos = torch.tensor([0, 5, 63], device="cuda")
    x, w = _randn(3, 2, 32, seed=4), _randn(3, 2, 32, seed=5)
    grad = serving.rotary(w, None, pos, table, layout=layout, inverse=True)[0]
    x64 = x.double().requires_grad_()
    (_turn64(x64, pos, table, layout) * w.double()).sum().backward()
    assert ((grad.double() - x64.grad).abs() <= _rot_tol(x64.grad, 2.0**-22)).all()
    for at in [(0, 0, 0), (1, 1, 13), (2, 0, 23), (2, 1, 31)]:
        step = torch.zeros_like(x)
        step[at] = 1.0
        hi, lo = serving.rotary(x + step, None, pos, table, layout=layout)[0], serving.rotary(x - step, None, pos, table, layout=layout)[0]
        slope = ((hi.double() - lo.double()) * w.double()).sum() / 2
        assert abs(slope - grad[at]) <= 32 * 2.0**-22 * 8  # 32 terms of at most 8 each in size


@pytest.mark.parametrize("scaling,more", [(None, {}), ("linear", dict(factor=4.0)), ("base", dict(factor=8.0)),
                                          ("ramp", dict(factor=8.0, original=4096, magnitude=1.2))])
def test_rotary_table(scaling, more):
    table = serving.rotary_table(64, 40000, base=10000.0, scaling=scaling, **more)
    f, mag = more.get("factor", 1.0), more.get("magnitude", 1.0)
    for i in (0, 1, 7, 19, 31):
        theta = 10000.0 ** (-2 * i / 64)
        if scaling == "linear":
            theta /= f
        if scaling == "base":
            theta = (10000.0 * f ** (64 / 62)) ** (-2 * i / 64)
        if scaling == "ramp":
            keep = min(1.0, max(0.0, (4096 * theta / (2 * math.pi) - 1) / 31))
            theta = theta * keep + theta / f * (1 - keep)
        for pos in (0, 1, 1000, 39999):
            # the angle in 64 bits is off by at most 40000 * 2^-50
            assert abs(table[pos, i].item() - mag * math.cos(pos * theta)) < 2e-7
            assert abs(table[pos, 32 + i].item() - mag * math.sin(pos * theta)) < 2e-7


# ---- the cache -------------------------------------------------------------------------------------


def _quantised(x, dtype):
    """(codes, scales) of rows, in f32 with IEEE operations as documented."""
    x = x.float()
    scale = x.abs().amax(-1) / torch.tensor(TOP[dtype], device="cuda")
    y = torch.where(scale[..., None] > 0, x / scale[..., None], 0.0)
    return (y.round().to(torch.int8) if dtype == "i8" else y.to(torch.float8_e4m3fn)), scale


def _at(cache, slots):
    return slots.long() // cache.page_size, slots.long() % cache.page_size


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "i8", "e4m3"])
@pytest.mark.parametrize("tokens,heads,dim,page,source", [(1, 1, 8, 1, "f32"), (3, 8, 128, 16, "bf16"), (70, 3, 80, 24, "f16"),
                                                          (257, 2, 96, 7, "f32"), (19, 5, 512, 3, "bf16"), (130, 1, 72, 64, "f16")])
def test_cache_write_and_read(heads_first, dtype, tokens, heads, dim, page, source):
    pages = -(-tokens // page) + 2
    cache = serving.PagedCache.empty(pages, page, heads, dim, dtype, heads_first=heads_first)
    before = serving.cache_read(cache, torch.arange(pages * page, device="cuda"), "f32")
    k, v = _randn(tokens, heads, dim, dtype=DT[source], seed=1, scale=3.0), _randn(tokens, heads, dim, dtype=DT[source], seed=2)
    k[0, 0] = 0.0
    slots = torch.randperm(pages * page, device="cuda", generator=_gen(3))[:tokens].int()
    slots[tokens // 2] = -1
    serving.cache_write(cache, k, v, slots)
    live = slots >= 0
    for x, pool, scales, back in zip((k, v), (cache.k, cache.v), (cache.k_scale, cache.v_scale), serving.cache_read(cache, slots, "f32")):
        got = pool[_at(cache, slots[live])]
        if dtype in TOP:
            codes, scale = _quantised(x[live], dtype)
            assert torch.equal(got.view(torch.int8), codes.view(torch.int8))
            assert torch.equal(scales[_at(cache, slots[live])], scale)
            want = codes.float() * scale[..., None]
            # a code is off by half a step at most
            step = scale[..., None] * (0.5 if dtype == "i8" else 16.0)
            assert ((want - x[live].float()).abs() <= step * 1.0001).all()
        else:
            want = x[live].to(DT[dtype])
            assert torch.equal(got, want)
        assert torch.equal(back[live], want.float()) and (back[~live] == 0).all()
        for out in ("f16", "bf16"):
            half = serving.cache_read(cache, slots, out)[0 if x is k else 1]
            assert torch.equal(half[live], want.float().to(DT[out]))
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[live].long()] = False
    for a, b in zip(before, serving.cache_read(cache, torch.arange(pages * page, device="cuda"), "f32")):
        assert torch.equal(a[rest], b[rest])


def test_cache_write_of_what_is_not_finite():
    cache = serving.PagedCache.empty(2, 4, 2, 16, "i8")
    k = torch.ones(3, 2, 16, device="cuda")
    k[0, 0, 3], k[1, 1, 5], k[2, 0, 0] = math.inf, math.nan, 1e-42
    v = torch.full((3, 2, 16), 3.0e38, device="cuda")
    v[1] = 1e-45
    serving.cache_write(cache, k, v, torch.tensor([0, 5, 2], device="cuda"))
    back, vback = serving.cache_read(cache, torch.tensor([0, 5, 2], device="cuda"), "f32")
    assert back[0, 0].isnan().all() and (back[0, 1] == 1).all() and back[1, 1].isnan().all() and (back[2] <= 1).all()
    assert ((vback[0] / 3.0e38 - 1).abs() < 1e-6).all() and vback.isfinite().all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["bf16", "i8", "e4m3"])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot", [(1, 32, 8, 128, 128), (50, 3, 2, 96, 40), (9, 4, 4, 64, 64), (300, 7, 1, 128, 64)])
def test_rotary_cache_write_is_both(layout, dtype, tokens, hq, hk, dim, rot):
    table = serving.rotary_table(rot, 1000)
    rows = _randn(tokens, hq + 2 * hk, dim, dtype=torch.bfloat16, seed=6)
    q, k, v = rows[:, :hq], rows[:, hq : hq + hk], rows[:, hq + hk :]
    pos = torch.randint(0, 1000, (tokens,), device="cuda", generator=_gen(7))
    slots = torch.randperm(320, device="cuda", generator=_gen(8))[:tokens]
    one, two = (serving.PagedCache.empty(20, 16, hk, dim, dtype) for _ in range(2))
    got = serving.rotary_cache_write(one, q, k, v, slots, pos, table, layout=layout)
    q2, _ = serving.rotary(q, None, pos, table, layout=layout)
    turned, _ = serving.rotary(k.float(), None, pos, table, layout=layout)  # not rounded before it is quantised
    serving.cache_write(two, turned, v.float(), slots)
    assert torch.equal(got, q2)
    for a, b in ((one.k, two.k), (one.v, two.v), (one.k_scale, two.k_scale), (one.v_scale, two.v_scale)):
        assert a is None or torch.equal(a.view(torch.int8) if a.element_size() == 1 else a, b.view(torch.int8) if b.element_size() == 1 else b)
    assert serving.rotary_cache_write(one, None, k, v, slots, pos, table, layout=layout) is None


# ---- attention -------------------------------------------------------------------------------------


def _case(lens, hq, hk, dim, dtype="bf16", cache_dtype="bf16", page=16, heads_first=False, seed=0, scale=1.0, junk=True):
    """A filled cache and queries for [(new, context), ...]; what no token may see is NaN or a bad page."""
    need = sum(-(-c // page) for _, c in lens)
    cache = serving.PagedCache.empty(need + 3, page, hk, dim, cache_dtype, heads_first=heads_first)
    if junk:
        if cache_dtype in TOP:
            cache.k_scale.fill_(math.nan), cache.v_scale.fill_(math.nan)
        else:
            cache.k.fill_(math.nan), cache.v.fill_(math.nan)
    order = torch.randperm(need + 3, device="cuda", generator=_gen(seed))
    wide = max(1, max(-(-c // page) for _, c in lens)) + 2
    table = torch.full((len(lens), wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, (_, c) in enumerate(lens):
        n = -(-c // page)
        table[b, :n] = order[at : at + n]
        at += n
        if c:
            key = torch.arange(c, device="cuda")
            slots = table[b].long()[key // page] * page + key % page
            serving.cache_write(cache, _randn(c, hk, dim, seed=seed * 100 + 2 * b + 1, scale=scale),
                                _randn(c, hk, dim, seed=seed * 100 + 2 * b + 2), slots)
    tokens = sum(n for n, _ in lens)
    q = _randn(tokens, hq, dim, dtype=DT[dtype], seed=seed + 50)
    starts = torch.tensor([0] + [n for n, _ in lens], device="cuda").cumsum(0).int()
    return q, cache, table, torch.tensor([c for _, c in lens], device="cuda", dtype=torch.int32), starts


def _attend64(q, cache, table, lens, starts, window=0, causal=True, scale=None):
    """(out, lse, sum of p |v|) in 64 bits."""
    hq, dim = q.shape[1:]
    group = hq // cache.kv_heads
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    size, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    scale = dim**-0.5 if scale is None else scale
    for b in range(table.shape[0]):
        n0, n1, c = int(starts[b]), int(starts[b + 1]), int(lens[b])
        n = n1 - n0
        if not n or not c:
            continue
        key = torch.arange(c, device="cuda")
        k, v = (x.double() for x in serving.cache_read(cache, table[b].long()[key // cache.page_size] * cache.page_size + key % cache.page_size, "f32"))
        place = torch.arange(c - n, c, device="cuda")[:, None]
        seen = key <= place if causal else torch.ones(n, c, dtype=torch.bool, device="cuda")
        if window:
            seen &= key > place - window
        s = torch.einsum("nhgd,lhd->hgnl", q[n0:n1].double().view(n, cache.kv_heads, group, dim), k) * scale
        s = s.masked_fill(~seen, -math.inf)
        row = torch.logsumexp(s, -1)
        p = torch.where(row[..., None] == -math.inf, 0.0, (s - row[..., None]).exp())
        o = torch.einsum("hgnl,lhd->nhgd", p, v).reshape(n, hq, dim)
        out[n0:n1], lse[n0:n1] = o, row.permute(2, 0, 1).reshape(n, hq)
        size[n0:n1] = torch.einsum("hgnl,lhd->nhgd", p, v.abs()).reshape(n, hq, dim)
    return out, lse, size


def _agree(case, max_new=None, decode=False, **how):
    q, cache, table, lens, starts = case
    out, lse = serving.paged_attention(q, cache, table, lens, None if decode else starts, max_new=max_new, return_lse=True, **how)
    want, want_lse, size = _attend64(q, cache, table, lens, starts, **how)
    u = U[q.dtype]
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    least = 2.0**-25 if q.dtype == torch.float16 else 0.0  # half of f16's smallest step: results below 2^-14
    off = (out.double() - want).abs() - (u * (want.abs() + size) + 2e-5 * size + least)
    assert (off <= 0).all(), f"{off.max().item()} over the bound at {(off == off.max()).nonzero()[0].tolist()}"
    assert torch.equal(lse == -math.inf, want_lse == -math.inf)
    fine = want_lse != -math.inf
    assert ((lse.double() - want_lse).abs()[fine] <= 2e-5 * want_lse.abs()[fine].clamp(min=1)).all()
    return out


FORMS = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "i8"), ("f16", "i8"), ("bf16", "e4m3"), ("f16", "e4m3")]


@pytest.mark.parametrize("dtype,cache_dtype", FORMS)
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 64), (8, 2, 128), (16, 16, 64), (14, 2, 64), (40, 2, 128)])
def test_single_tokens(dtype, cache_dtype, hq, hk, dim):
    lens = [(1, c) for c in (1, 2, 15, 16, 17, 127, 128, 129, 700, 2500)]
    _agree(_case(lens, hq, hk, dim, dtype, cache_dtype), decode=True)


@pytest.mark.parametrize("page,heads_first", [(1, False), (3, True), (8, False), (24, False), (64, True), (128, False), (256, True)])
@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
def test_pages_of_every_size(page, heads_first, cache_dtype):
    lens = [(1, 333), (1, 64), (1, 1)]
    _agree(_case(lens, 4, 2, 128, "bf16", cache_dtype, page, heads_first), decode=True)
    lens = [(40, 333), (1, 64), (3, 3), (130, 1000)]
    _agree(_case(lens, 4, 2, 128, "bf16", cache_dtype, page, heads_first, seed=1), max_new=130)


@pytest.mark.parametrize("dtype,cache_dtype", FORMS)
@pytest.mark.parametrize("hq,hk,dim", [(2, 2, 64), (8, 2, 128), (7, 1, 128), (10, 2, 64), (3, 3, 128)])
def test_chunks(dtype, cache_dtype, hq, hk, dim):
    lens = [(37, 37), (1, 900), (0, 50), (129, 400), (300, 301), (5, 0), (64, 640), (2, 128), (257, 1025)]
    _agree(_case(lens, hq, hk, dim, dtype, cache_dtype, seed=2), max_new=300)


@pytest.mark.parametrize("new", [1, 2, 4, 5, 16, 31, 32, 33, 64, 65, 128, 129, 200])
@pytest.mark.parametrize("cache_dtype", ["bf16", "e4m3"])
def test_chunk_lengths(new, cache_dtype):
    for max_new in (None, new):
        _agree(_case([(new, new), (new, new + 77), (1, 300)], 8, 2, 64, "bf16", cache_dtype, seed=3), max_new=max_new)


@pytest.mark.parametrize("window", [1, 2, 16, 100, 128, 129, 5000])
@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
def test_windows(window, cache_dtype):
    lens = [(1, 1), (1, 500), (60, 300), (200, 200), (9, 2000)]
    _agree(_case(lens, 6, 2, 128, "bf16", cache_dtype, seed=4), max_new=200, window=window)
    _agree(_case([(1, 1), (1, 130), (1, 3000)], 6, 2, 64, "bf16", cache_dtype, seed=5), decode=True, window=window)


@pytest.mark.parametrize("new", [3, 150])
def test_without_causal_mask(new):
    _agree(_case([(new, new), (new, 1000), (1, 7)], 4, 4, 64, seed=6), max_new=new, causal=False)


def test_rows_that_see_nothing():
    """More new tokens than keys (the first ones stand before the sequence's start), and sequences without keys."""
    for dim, lens in ((64, [(5, 2), (1, 0), (4, 4)]), (128, [(200, 150), (40, 0), (130, 1)])):
        case = _case(lens, 4, 2, dim, seed=7)
        out = _agree(case, max_new=max(n for n, _ in lens))
        assert (out[: lens[0][0] - lens[0][1]] == 0).all()
    _agree(_case([(1, 0), (1, 0)], 4, 2, 64, seed=8), decode=True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("cache_dtype", ["f16", "i8"])
@pytest.mark.parametrize("new", [1, 260])
def test_large_scores_and_uneven_scales(dim, cache_dtype, new):
    """Scores in the hundreds, growing along the keys, and value scales from 1e-6 to 1e3."""
    q, cache, table, lens, starts = _case([(new, 900), (new, new)], 4, 2, dim, "f16", cache_dtype, seed=9, scale=8.0)
    key = torch.arange(900, device="cuda")
    slots = table[0].long()[key // 16] * 16 + key % 16
    grow = torch.logspace(-6, 3 if cache_dtype == "i8" else 1, 900, device="cuda")[:, None, None]
    k = q[:1, :2].float() * (key / 60)[:, None, None]
    serving.cache_write(cache, k.contiguous(), _randn(900, 2, dim, seed=10) * grow, slots)
    _agree((q, cache, table, lens, starts), max_new=new)


def test_splits_of_long_contexts_and_large_batches():
    _agree(_case([(1, 70001)], 8, 1, 64, "bf16", "bf16", 16, seed=11), decode=True)
    _agree(_case([(17, 40000)], 4, 1, 128, "bf16", "i8", 64, seed=12), max_new=17)
    _agree(_case([(1, 1 + 37 * i % 600) for i in range(333)], 4, 2, 64, "f16", "f16", 16, seed=13), decode=True)
    _agree(_case([(1 + i % 9, 9 + 53 * i % 700) for i in range(150)], 4, 1, 128, "bf16", "e4m3", 16, seed=14), max_new=9)


@pytest.mark.parametrize("new", [1, 300])
def test_results_do_not_change_between_calls(new):
    q, cache, table, lens, starts = _case([(new, 9000), (1, 500)], 8, 2, 128, seed=15)
    first = serving.paged_attention(q, cache, table, lens, starts, max_new=new)
    for _ in range(5):
        assert torch.equal(first, serving.paged_attention(q, cache, table, lens, starts, max_new=new))


@pytest.mark.parametrize("new", [1, 140])
def test_strided_queries_outputs_and_wide_tables(new):
    q, cache, table, lens, starts = _case([(new, 200), (new, 333)], 4, 2, 64, seed=16)
    want = serving.paged_attention(q, cache, table, lens, starts, max_new=new)
    rows = torch.zeros(2 * new, 9, 64, dtype=q.dtype, device="cuda")
    rows[:, 2:6] = q
    wide = torch.full((2, 500), -7, dtype=torch.int64, device="cuda")
    wide[:, : table.shape[1]] = table
    out = torch.zeros(2 * new, 8, 64, dtype=q.dtype, device="cuda")
    got = serving.paged_attention(rows[:, 2:6], cache, wide, lens.long(), starts.long(), max_new=new, out=out[:, ::2])
    assert torch.equal(got, want) and (out[:, 1::2] == 0).all()
    odd = torch.zeros(2 * new, 4, 65, dtype=q.dtype, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(serving.paged_attention(odd, cache, table, lens, starts, max_new=new), want)
    assert serving.paged_attention(q[:0], cache, table, lens, starts * 0, max_new=1).shape == (0, 4, 64)
    # tokens that belong to no sequence are not written
    pad = torch.cat((q, q))
    out = torch.full(pad.shape, 3.0, dtype=q.dtype, device="cuda")
    serving.paged_attention(pad, cache, table, lens, starts, max_new=new, out=out)
    assert torch.equal(out[: 2 * new], want) and (out[2 * new :] == 3).all()


def test_streams_and_graphs():
    q, cache, table, lens, starts = _case([(1, 5000), (1, 300), (1, 80)], 8, 2, 128, seed=17)
    want = serving.paged_attention(q, cache, table, lens)
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s in side:
            with torch.cuda.stream(s):
                got.append(serving.paged_attention(q, cache, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = serving.paged_attention(q, cache, table, lens)
    for n in (5000, 77):
        lens[0] = n
        graph.replay()
        assert torch.equal(out, serving.paged_attention(q, cache, table, lens))


def test_what_the_device_refuses():
    """Indexes out of range are skipped and recorded, and the context stays usable."""
    q, cache, table, lens, starts = _case([(1, 100), (1, 40)], 4, 2, 64, seed=18)
    want = serving.paged_attention(q, cache, table, lens)
    serving.check()
    bad = table.clone()
    bad[1, 0] = cache.pages
    got = serving.paged_attention(q, cache, bad, lens)
    with pytest.raises(rt.RuntimeError_, match="paged_attention: page"):
        serving.check()
    assert torch.equal(got[0], want[0])
    serving.paged_attention(q, cache, table[:, :3].contiguous(), lens)
    with pytest.raises(rt.RuntimeError_, match="paged_attention: length"):
        serving.check()
    rows = _randn(2, 2, 64, dtype=torch.bfloat16)
    held = cache.k.clone()
    serving.cache_write(cache, rows, rows, torch.tensor([cache.pages * 16, -1], device="cuda"))
    with pytest.raises(rt.RuntimeError_, match="cache_write: slot"):
        serving.check()
    assert torch.equal(cache.k.nan_to_num(9.0), held.nan_to_num(9.0))
    serving.cache_read(cache, torch.tensor([cache.pages * 16], device="cuda"))
    with pytest.raises(rt.RuntimeError_, match="cache_read: slot"):
        serving.check()
    turned, _ = serving.rotary(rows, None, torch.tensor([3, 4096], device="cuda"), serving.rotary_table(64, 4096))
    with pytest.raises(rt.RuntimeError_, match="rotary: position"):
        serving.check()
    assert turned[0].isfinite().all() and turned[1].isnan().all()
    serving.check()


def test_what_is_refused_before_a_launch():
    def full(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    cache = serving.PagedCache.empty(4, 16, 2, 64)
    for how, why in [((full(4, 16, 2, 64), full(4, 16, 2, 32)), "same shape"), ((full(4, 16, 2, 60), full(4, 16, 2, 60)), "multiple of 8"),
                     ((full(4, 16, 2, 64), full(4, 2, 16, 64).transpose(1, 2)), "same shape and strides"),
                     ((full(4, 16, 2, 64), full(4, 16, 2, 64, dtype=torch.float16)), "dtype"),
                     ((full(4, 16, 2, 65)[..., 1:], full(4, 16, 2, 65)[..., 1:]), "boundaries"),
                     ((full(4, 16, 2, 64, dtype=torch.int8), full(4, 16, 2, 64, dtype=torch.int8)), "needs k_scale"),
                     ((full(4, 16, 2, 64), full(4, 16, 2, 64), full(4, 16, 2), full(4, 16, 2)), "no scales"),
                     ((full(4, 16, 2, 64, dtype=torch.int8), full(4, 16, 2, 64, dtype=torch.int8), full(4, 16, 1, dtype=torch.float32),
                       full(4, 16, 2, dtype=torch.float32)), "expected shape")]:
        with pytest.raises(ValueError, match=why):
            serving.PagedCache(*how)
    x, slots, table = full(3, 2, 64), torch.zeros(3, dtype=torch.int32, device="cuda"), serving.rotary_table(64, 8)
    for call, why in [(lambda: serving.cache_write(cache, full(3, 1, 64), full(3, 1, 64), slots), "do not go with"),
                      (lambda: serving.cache_write(cache, x, x, slots[:2]), "expected 3 entries"),
                      (lambda: serving.cache_write(cache, x, x.float(), slots), "dtype"),
                      (lambda: serving.cache_read(cache, slots.float()), "dtype"),
                      (lambda: serving.cache_read(cache, slots, "i8"), "dtype must be"),
                      (lambda: serving.rotary(x, None, slots, table, layout="other"), "layout"),
                      (lambda: serving.rotary(x, None, slots, full(8, 66, dtype=torch.float32)), "do not turn"),
                      (lambda: serving.rotary(x, full(2, 2, 64), slots, table), "does not go with"),
                      (lambda: serving.rotary(x, None, slots, table, out=(full(3, 2, 32), None)), "expected shape"),
                      (lambda: serving.rotary_cache_write(cache, full(3, 2, 32), x, x, slots, slots, table), "does not go with")]:
        with pytest.raises(ValueError, match=why):
            call()
    with pytest.raises(TypeError):
        serving.rotary_cache_write(cache, x, x, x, slots, None, None)
    pages, lens = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), slots
    for call, why in [(lambda: serving.paged_attention(full(3, 3, 64), cache, pages, lens), "does not go with"),
                      (lambda: serving.paged_attention(full(3, 2, 64, dtype=torch.float16), cache, pages, lens), "must have q's dtype"),
                      (lambda: serving.paged_attention(full(3, 2, 96), serving.PagedCache.empty(4, 16, 2, 96), pages, lens), "64 or 128"),
                      (lambda: serving.paged_attention(full(4, 2, 64), cache, pages, lens), "one token to a sequence"),
                      (lambda: serving.paged_attention(x, cache, pages, lens, lens), "expected 4 entries"),
                      (lambda: serving.paged_attention(x, cache, pages[:, :0], lens), "no columns"),
                      (lambda: serving.paged_attention(x, cache, pages, lens, window=-1), "window"),
                      (lambda: serving.paged_attention(x, cache, pages, lens, max_new=0), "max_new"),
                      (lambda: serving.paged_attention(x, cache, pages, lens, scale=0.0), "scale"),
                      (lambda: serving.paged_attention(x.float(), cache, pages, lens), "dtype")]:
        with pytest.raises(ValueError, match=why):
            call()


@pytest.mark.parametrize("new", [1, 300])
@pytest.mark.parametrize("cache_dtype,dim", [("i8", 128), ("e4m3", 64)])
def test_very_small_values_beside_zeros(new, cache_dtype, dim):
    """Value scales around 1e-16, and every third key's scale 0: nothing is held at a larger size."""
    case = _case([(new, 700), (new, 333), (new, new)], 8, 2, dim, "bf16", cache_dtype, seed=21)
    scale = case[1].v_scale
    scale.mul_(1e-15)
    scale.view(-1, scale.shape[-1])[::3] = 0
    _agree(case, max_new=new)


@pytest.mark.parametrize("new", [1, 300])
def test_a_value_row_held_as_nan_reaches_the_output(new):
    case = _case([(new, 700)], 8, 2, 128, "bf16", "i8", seed=22)
    q, cache, table, lens, starts = case
    cache.v_scale[table[0, 0].item(), 3] = math.nan
    out = serving.paged_attention(q, cache, table, lens, starts, max_new=new)
    assert out.isnan().all()


@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
@pytest.mark.parametrize("hq,hk,dim,new,max_new,window", [(1, 1, 64, 300, 300, 16), (1, 1, 64, 300, 300, 100), (32, 8, 128, 60, 1, 7),
                                                          (8, 2, 128, 500, 500, 129), (4, 4, 64, 700, 1, 300)])
def test_windows_without_causal_mask(hq, hk, dim, new, max_new, window, cache_dtype):
    """Without the causal mask a window hides only what is before it, so a tile's keys go on to the sequence's end.  (max_new
    chooses the kernel and nothing else: 1 gives the kernel of few rows.)  A cut call after it on the same
    stream finds its counters at zero."""
    lens = [(new, 1000), (3, 700), (new, new), (1, 2000)]
    plain = _case([(1, 9000), (2, 3000)], hq, hk, dim, "bf16", cache_dtype, seed=31)
    want = [_agree(plain, max_new=2) for _ in range(2)]
    _agree(_case(lens, hq, hk, dim, "bf16", cache_dtype, seed=30), max_new=max_new, window=window, causal=False)
    _agree(_case(lens[:1], hq, hk, dim, "bf16", cache_dtype, seed=32), max_new=max_new, window=window, causal=False)
    for _ in range(3):
        assert torch.equal(_agree(plain, max_new=2), want[0])


@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 2**63 - 1])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
def test_windows_as_long_as_integers_go(window, causal, cache_dtype):
    case = _case([(1, 1), (1, 5000), (1, 130)], 8, 2, 128, "bf16", cache_dtype, seed=33)
    _agree(case, decode=True, window=window, causal=causal)
    case = _case([(200, 200), (1, 5000), (90, 3000)], 8, 2, 128, "bf16", cache_dtype, seed=34)
    _agree(case, max_new=200, window=window, causal=causal)


@pytest.mark.parametrize("new,max_new", [(40, 1), (300, 300)])
@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
def test_token_ranges_out_of_order_or_range(new, max_new, cache_dtype):
    """Descending q_starts: nothing is written and the fault is recorded; beyond q: the rows that there are, and a
    record.  A cut call after it on the same stream finds its counters at zero.  (max_new 1: the kernel of few rows.)"""
    q, cache, table, lens, starts = _case([(new, 3000), (new, 4000), (new, 3500), (new, 2500)], 8, 2, 64, "bf16", cache_dtype, seed=35)
    good = serving.paged_attention(q, cache, table, lens, starts, max_new=max_new)
    serving.check()
    for bad in ([0, 4 * new, 0, 4 * new, 0], [0, new, new, 3 * new, 2 * new], [7, 6, 7, 8, 9]):
        out = torch.full_like(q, 3.0)
        serving.paged_attention(q, cache, table, lens, torch.tensor(bad, device="cuda"), max_new=max_new, out=out)
        with pytest.raises(rt.RuntimeError_, match="paged_attention: q_starts"):
            serving.check()
        assert (out == 3.0).all()
    for _ in range(3):
        assert torch.equal(serving.paged_attention(q, cache, table, lens, starts, max_new=max_new), good)
    long = torch.tensor([-3, new, 2 * new, 3 * new, 4 * new + 9], device="cuda")
    got = serving.paged_attention(q, cache, table, lens, long, max_new=max_new)
    with pytest.raises(rt.RuntimeError_, match="paged_attention: q_starts"):
        serving.check()
    assert torch.equal(got, good)


@pytest.mark.parametrize("wrap", [2**32, -(2**32), 2**62])
def test_64_bit_indices_do_not_wrap(wrap):
    """An index whose low half is valid is out of range all the same: skipped and recorded, negative slots skipped."""
    cache = serving.PagedCache.empty(4, 16, 2, 64, "bf16")
    x = _randn(3, 2, 64, dtype=torch.bfloat16)
    slots = torch.tensor([[7, 0], [5 + wrap, 0], [9, 0]], device="cuda")[:, 0]  # strided too
    serving.cache_write(cache, x, x, slots)
    if wrap > 0:
        with pytest.raises(rt.RuntimeError_, match="cache_write: slot"):
            serving.check()
    assert torch.equal(cache.k[0, 7], x[0]) and torch.equal(cache.v[0, 9], x[2]) and (cache.k[0, 5] == 0).all()
    cache.k[0, 5] = 1.0
    back = serving.cache_read(cache, slots)[0]
    if wrap > 0:
        with pytest.raises(rt.RuntimeError_, match="cache_read: slot"):
            serving.check()
    assert torch.equal(back[0], x[0]) and (back[1] == 0).all() and torch.equal(back[2], x[2])
    turned, _ = serving.rotary(x, None, slots, serving.rotary_table(64, 16))
    with pytest.raises(rt.RuntimeError_, match="rotary: position"):
        serving.check()
    assert turned[0].isfinite().all() and turned[1].isnan().all() and turned[2].isfinite().all()
    case = _case([(1, 100), (1, 40)], 4, 2, 64, seed=36)
    q, cache, table, lens, starts = case
    want = serving.paged_attention(q, cache, table, lens)
    wide = torch.stack((table.long(), table.long()), 2)[..., 1]
    assert torch.equal(serving.paged_attention(q, cache, wide, lens.long(), starts.long(), max_new=1), want)
    for what in ("page", "length", "q_starts"):
        t, n, s = table.long(), lens.long(), starts.long()
        if what == "page":
            t[1, 0] += wrap
        elif what == "length":
            n[1] += wrap
        else:
            s[2] += wrap
        got = serving.paged_attention(q, cache, t, n, s, max_new=1)
        with pytest.raises(rt.RuntimeError_, match=f"paged_attention: {what}"):
            serving.check()
        assert (what == "q_starts" and wrap < 0) or torch.equal(got[0], want[0])


@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
def test_single_tokens_without_max_new_take_the_kernel_of_few_rows(cache_dtype):
    """q_starts alone do not say how many new tokens a sequence has; single tokens are still not planned as if each
    had all of them, so the bits are those of the call without q_starts.  With max_new given, rows of no sequence
    change no bit."""
    q, cache, table, lens, starts = _case([(1, 100 + 61 * i) for i in range(64)], 32, 8, 128, "bf16", cache_dtype, seed=37)
    want = serving.paged_attention(q, cache, table, lens)
    assert torch.equal(serving.paged_attention(q, cache, table, lens, starts), want)
    for new in (1, 33, 64):
        case = _case([(new, 900), (1, 400)], 32, 8, 128, "bf16", cache_dtype, seed=38)
        _agree(case)
        q, cache, table, lens, starts = case
        want = serving.paged_attention(q, cache, table, lens, starts, max_new=new)
        padded = serving.paged_attention(torch.cat((q, q[:1].expand(70, -1, -1))), cache, table, lens, starts, max_new=new)
        assert torch.equal(padded[: new + 1], want)


@pytest.mark.parametrize("factor", [2.0**40, 2.0**-60, 2.0**120, math.inf, math.nan])
@pytest.mark.parametrize("cache_dtype,dim", [("i8", 128), ("e4m3", 64), ("bf16", 128)])
@pytest.mark.parametrize("max_new", [1, 200])
def test_a_token_of_another_size_does_not_reach_the_others(factor, cache_dtype, dim, max_new):
    """Rows of other tokens and heads share a tile: however large, small or broken one token's query is, or one head's, the
    others' results do not know.  (max_new 1: the kernel of few rows.)"""
    q, cache, table, lens, starts = _case([(3, 500), (1, 333), (5, 5), (40, 700), (200, 900)], 8, 2, dim, "bf16", cache_dtype, seed=40)
    q[1] *= factor
    q[3, 2] *= factor
    q[12, :, 3] *= factor
    plain = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    if factor > 1 or factor != factor:
        plain[1], plain[3, 2], plain[12] = False, False, False
    out, lse = serving.paged_attention(q, cache, table, lens, starts, max_new=max_new, return_lse=True)
    want, want_lse, size = _attend64(q, cache, table, lens, starts)
    off = (out.double() - want).abs() - (U[q.dtype] * (want.abs() + size) + 2e-5 * size)
    assert (off[plain] <= 0).all(), off[plain].max().item()
    assert ((lse.double() - want_lse).abs()[plain] <= 2e-5 * want_lse.abs()[plain].clamp(min=1)).all()
    if not math.isfinite(factor):
        assert out[1].isnan().all()


def _top_scores64(q, cache, table, lens, starts):
    """Each row's largest score and its distance to the next, of a causal call in 64 bits."""
    hq, dim = q.shape[1:]
    top = torch.full((*q.shape[:2], 2), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(table.shape[0]):
        n0, n1, c = int(starts[b]), int(starts[b + 1]), int(lens[b])
        key = torch.arange(c, device="cuda")
        k = serving.cache_read(cache, table[b].long()[key // cache.page_size] * cache.page_size + key % cache.page_size, "f32")[0].double()
        s = torch.einsum("nhd,lhd->nhl", q[n0:n1].double(), k.repeat_interleave(hq // cache.kv_heads, 1)) * dim**-0.5
        top[n0:n1] = s.masked_fill((key > torch.arange(c - n1 + n0, c, device="cuda")[:, None])[:, None], -math.inf).topk(2, -1).values
    return top[..., 0], top[..., 0] - top[..., 1]


@pytest.mark.parametrize("dtype,cache_dtype,grow,scale", [("bf16", "bf16", 2.0**40, 16.0), ("bf16", "i8", 2.0**40, 16.0), ("bf16", "e4m3", 2.0**30, 16.0),
                                                          ("f16", "f16", 2.0**13, 4e3), ("f16", "i8", 2.0**13, 4e3), ("bf16", "bf16", 2.0**12, 16.0)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("max_new", [1, 300])
def test_scores_past_what_f32_tells_apart(dtype, cache_dtype, grow, scale, dim, max_new):
    """Scores of 2^18 to 2^46 in every third row.  A score's f32 error is at most 128 2^-24 of its products' sizes, which
    come to some 11 times the largest score's: 2^-13 of it.  Rows whose largest score is further than twice that and
    50 above the next have that key's value; in rows with scores under 300 the usual bound holds; all are finite."""
    q, cache, table, lens, starts = _case([(300, 900), (3, 333), (260, 260)], 4, 2, dim, dtype, cache_dtype, seed=42, scale=scale)
    q[::3] *= grow
    out, lse = serving.paged_attention(q, cache, table, lens, starts, max_new=max_new, return_lse=True)
    want, want_lse, size = _attend64(q, cache, table, lens, starts)
    top, gap = _top_scores64(q, cache, table, lens, starts)
    sure = (gap > 50 + 2.0**-12 * top.abs()) | (top.abs() < 300)
    assert out.isfinite().all() and lse.isfinite().all() and sure[::3].any() and top.max() > 2.0**18
    off = (out.double() - want).abs() - (U[q.dtype] * (want.abs() + size) + 2e-5 * size + 2.0**-25)
    assert (off[sure] <= 0).all()
    assert ((lse.double() - want_lse).abs() <= 2.0**-13 * want_lse.abs().clamp(min=1)).all()


def test_every_code_reads_as_its_value():
    """All 256 codes of a borrowed 8-bit cache, e4m3's two NaN among them."""
    codes = torch.arange(256, device="cuda").to(torch.uint8).view(1, 2, 1, 128)
    for dtype in ("i8", "e4m3"):
        k = codes.view(DT[dtype])
        scale = torch.tensor([0.5, 3.0], device="cuda").view(1, 2, 1)
        cache = serving.PagedCache(k, k.clone(), scale, scale)
        want = k.float().view(2, 1, 128) * scale.view(2, 1, 1)
        for kind in ("f32", "f16", "bf16"):
            for got in serving.cache_read(cache, torch.arange(2, device="cuda"), kind):
                assert torch.equal(got.isnan(), want.isnan())
                assert torch.equal(got.nan_to_num(1e4), want.to(DT[kind]).nan_to_num(1e4))
        assert want.isnan().sum() == (2 if dtype == "e4m3" else 0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 300])
def test_nan_codes_reach_the_output(new, dim, dtype):
    q, cache, table, lens, starts = _case([(new, 700), (new, 333)], 8, 2, dim, dtype, "e4m3", seed=41)
    want = serving.paged_attention(q, cache, table, lens, starts, max_new=new)
    page, slot = table[0, 2].item(), 5
    for pool, code in ((cache.k, 0x7F), (cache.v, 0x7F), (cache.k, 0xFF), (cache.v, 0xFF)):
        held = pool[page, slot, 1, 9].clone()
        pool.view(torch.uint8)[page, slot, 1, 9] = code
        out = serving.paged_attention(q, cache, table, lens, starts, max_new=new)
        pool[page, slot, 1, 9] = held
        hit = out[:new, 4:] if pool is cache.k else out[:new, 4:, 9]
        assert hit.isnan().all()
        assert torch.equal(out[new:], want[new:]) and torch.equal(out[:new, :4], want[:new, :4])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_autograd_follows_rotary(layout, dtype):
    """d/dx <w, rotary(x)> through torch's graph, of q and of k, against 64-bit autograd; a table's magnitude, a second
    derivative (the map is linear: the gradient with respect to w turns back), an expanded gradient."""
    table = serving.rotary_table(24, 64, magnitude=1.25)
    pos = torch.tensor([0, 5, 63], device="cuda")
    x = [_randn(3, h, 32, dtype=DT[dtype], seed=4 + h).requires_grad_() for h in (4, 2)]
    w = [_randn(3, h, 32, dtype=DT[dtype], seed=14 + h).requires_grad_() for h in (4, 2)]
    got = serving.rotary(*x, pos, table, layout=layout)
    with torch.no_grad():
        plain = serving.rotary(*x, pos, table, layout=layout)
    assert all(torch.equal(a, b) and a.requires_grad and not b.requires_grad for a, b in zip(got, plain))
    grads = torch.autograd.grad(got, x, w, create_graph=True)
    u = 2.0**-22 if dtype == "f32" else U[DT[dtype]]
    for a, g, s in zip(x, grads, w):
        a64 = a.detach().double().requires_grad_()
        (_turn64(a64, pos, table, layout) * s.detach().double()).sum().backward()
        assert g.dtype == a.dtype and ((g.double() - a64.grad).abs() <= _rot_tol(a64.grad, u) * 1.6).all()
    again = torch.autograd.grad(grads, w, [a.detach() for a in x])
    assert all(torch.equal(a, b) for a, b in zip(again, plain))
    alone = serving.rotary(x[0], None, pos, table, layout=layout)
    assert alone[1] is None
    alone[0].sum().backward()
    ones = serving.rotary(torch.ones_like(x[0]).detach(), None, pos, table, layout=layout, inverse=True)[0]
    assert torch.equal(x[0].grad, ones) and x[1].grad is None
    cache = serving.PagedCache.empty(2, 4, 2, 32, "bf16")
    x[0].grad = None
    turned = serving.rotary_cache_write(cache, x[0], x[1], x[1], torch.arange(3, device="cuda"), pos, table, layout=layout)
    assert torch.equal(turned, plain[0])
    turned.sum().backward()
    assert torch.equal(x[0].grad, ones) and torch.equal(cache.v[0, :3], x[1].to(torch.bfloat16))


def test_what_has_no_gradient_says_so():
    """A result that would lose its gradient without a word is refused, at the latest in the backward pass."""
    q, cache, table, lens, starts = _case([(1, 100), (1, 40)], 4, 2, 64, seed=43)
    want = serving.paged_attention(q, cache, table, lens, return_lse=True)
    q.requires_grad_()
    got = serving.paged_attention(q, cache, table, lens, return_lse=True)
    assert all(torch.equal(a, b) and a.requires_grad for a, b in zip(got, want))
    with pytest.raises(NotImplementedError, match="no gradient"):
        got[0].sum().backward()
    with pytest.raises(NotImplementedError, match="no gradient"):
        serving.paged_attention(q, cache, table, lens).sum().backward()
    turns, pos = serving.rotary_table(64, 8), torch.zeros(2, dtype=torch.int32, device="cuda")
    for call in (lambda: serving.paged_attention(q, cache, table, lens, out=torch.empty_like(q)),
                 lambda: serving.rotary(q, None, pos, turns, out=(torch.empty_like(q), None)),
                 lambda: serving.rotary_cache_write(cache, q, q[:, :2], q[:, :2], pos - 1, pos, turns, out=torch.empty_like(q))):
        with pytest.raises(ValueError, match="require gradients"):
            call()
        with torch.no_grad():
            call()
    with pytest.raises(ValueError, match="table: no gradient"):
        serving.rotary(q, None, pos, turns.clone().requires_grad_())


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_a_cache_whose_memory_was_exchanged_is_refused(name):
    cache = serving.PagedCache.empty(4, 16, 2, 64, "i8")
    rows, slots = _randn(2, 2, 64), torch.arange(2, device="cuda")
    serving.cache_write(cache, rows, rows, slots)
    held = getattr(cache, name)
    kept = held.data
    held.data = held.clone()
    q, page, lens = _randn(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for call in (lambda: serving.cache_write(cache, rows, rows, slots), lambda: serving.cache_read(cache, slots),
                 lambda: serving.paged_attention(q, cache, page, lens)):
        with pytest.raises(ValueError, match="other memory"):
            call()
    held.data = kept
    serving.cache_write(cache, rows, rows, slots)


def test_changes_in_place_are_counted():
    """What autograd has kept for a backward pass and an operator then changes is noticed there."""
    q, cache, table, lens, starts = _case([(1, 100), (1, 40)], 4, 2, 64, "bf16", "i8", seed=44)
    half = serving.PagedCache.empty(4, 16, 2, 64, "bf16")
    turns, pos, slots = serving.rotary_table(64, 8), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.arange(2, device="cuda")
    rows, out, out2 = _randn(2, 2, 64, dtype=torch.bfloat16), torch.zeros_like(q), torch.zeros_like(q)
    for kept, call in ((half.k, lambda: serving.cache_write(half, rows, rows, slots)), (half.v, lambda: serving.cache_write(half, rows, rows, slots)),
                       (cache.k_scale, lambda: serving.cache_write(cache, rows, rows, slots)), (cache.v_scale, lambda: serving.cache_write(cache, rows, rows, slots)),
                       (half.k, lambda: serving.rotary_cache_write(half, None, rows, rows, slots, pos, turns)),
                       (out, lambda: serving.paged_attention(q, cache, table, lens, out=out)), (out, lambda: serving.rotary(q, None, pos, turns, out=(out, None))),
                       (out2, lambda: serving.rotary_cache_write(cache, q, rows, rows, slots, pos, turns, out=out2))):
        before = kept._version
        y = (torch.ones_like(kept, requires_grad=True) * kept).sum()
        call()
        assert kept._version == before + 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    leaf = serving.PagedCache(half.k.clone().requires_grad_(), half.v.clone())
    with pytest.raises(ValueError, match="requires gradients"):
        serving.cache_write(leaf, rows, rows, slots)
    with torch.no_grad():
        serving.cache_write(leaf, rows, rows, slots)
    with torch.inference_mode():
        made = serving.PagedCache.empty(4, 16, 2, 64, "bf16")
    serving.cache_write(made, rows, rows, slots)
    assert torch.equal(made.k[0, :2], rows) and torch.equal(leaf.v[0, :2], rows)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_more_heads_than_16_bits_count(layout):
    """140000 heads of one token: as the same rows of 140 tokens."""
    table, x = serving.rotary_table(264, 16), _randn(1, 140000, 264, dtype=torch.bfloat16)
    got, _ = serving.rotary(x, None, torch.tensor([7], device="cuda"), table, layout=layout)
    want, _ = serving.rotary(x.view(140, 1000, 264), None, torch.full((140,), 7, device="cuda"), table, layout=layout)
    assert torch.equal(got.view(-1), want.view(-1))


@pytest.mark.parametrize("new,max_new", [(1, 1), (300, 300)])
@pytest.mark.parametrize("cache_dtype", ["bf16", "i8"])
@pytest.mark.parametrize("page", [-1, -(2**31), 2**31 - 1])
def test_every_page_out_of_range_is_recorded(page, cache_dtype, new, max_new):
    q, cache, table, lens, starts = _case([(new, 900), (new, 500)], 8, 2, 64, "bf16", cache_dtype, seed=45)
    want = serving.paged_attention(q, cache, table, lens, starts, max_new=max_new)
    serving.check()
    table[1, 3] = page
    got = serving.paged_attention(q, cache, table, lens, starts, max_new=max_new)
    with pytest.raises(rt.RuntimeError_, match="paged_attention: page"):
        serving.check()
    assert torch.equal(got[:new], want[:new]) and got.isfinite().all()


def test_arguments_that_do_not_convert():
    """Python's own errors come through (text that is no text in UTF-8 ended the process)."""
    cache, x = serving.PagedCache.empty(4, 16, 2, 64), _randn(2, 2, 64, dtype=torch.bfloat16)
    slots, table = torch.zeros(2, dtype=torch.int32, device="cuda"), serving.rotary_table(64, 8)

    class Neither:
        def __bool__(self):
            raise ArithmeticError("neither")

    for call in (lambda: serving.rotary(x, None, slots, table, inverse=Neither()), lambda: serving.paged_attention(x, cache, slots[:, None], slots, causal=Neither()),
                 lambda: serving.paged_attention(x, cache, slots[:, None], slots, return_lse=Neither())):
        with pytest.raises(ArithmeticError, match="neither"):
            call()
    for call in (lambda: serving.rotary(x, None, slots, table, layout="\ud800"), lambda: serving.cache_read(cache, slots, "\ud800")):
        with pytest.raises(UnicodeEncodeError):
            call()
    for call in (lambda: serving.paged_attention(x, cache, slots[:, None], slots, max_new="x"), lambda: serving.paged_attention(x, cache, slots[:, None], slots, window=1.5),
                 lambda: serving.paged_attention(x, cache, slots[:, None], slots, scale="x")):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(OverflowError):
        serving.paged_attention(x, cache, slots[:, None], slots, window=2**63)


@pytest.mark.parametrize("new", [1, 300])
@pytest.mark.parametrize("dtype,top", [("bf16", 1e8), ("f16", 4e3)])
@pytest.mark.parametrize("cache_dtype", ["i8", "e4m3"])
def test_values_of_very_different_size_at_equal_scores(new, dtype, top, cache_dtype):
    """Every third key's values are as large as is promised (scales of 2^20; f16 results end at 65504), the others' small or
    zero, and all weigh the same."""
    case = _case([(new, 700), (new, 2000), (new, new)], 8, 2, 128, dtype, cache_dtype, seed=46)
    q, cache, table, lens, starts = case
    for b, c in enumerate(lens.tolist()):
        key = torch.arange(c, device="cuda")
        v = _randn(c, 2, 128, seed=47 + b) * torch.tensor([top / 4, 0.0, 1e-3], device="cuda")[key % 3][:, None, None]
        serving.cache_write(cache, _randn(c, 2, 128, seed=50 + b, scale=1e-6), v, table[b].long()[key // 16] * 16 + key % 16)
    _agree(case, max_new=new)


@pytest.mark.parametrize("dtype,cache_dtype", FORMS)
@pytest.mark.parametrize("new", [1, 260])
@pytest.mark.parametrize("dim", [64, 128])
def test_sharp_scores(dtype, cache_dtype, new, dim):
    """Scores 2 q k: probabilities down to e^-100, and elements that only improbable keys have (codes of 0).  Besides the usual
    bound, each of 400 keys is off by at most 2^-39 of its value where P is f16, and the scores' f32 error, for
    scores of some 100, is 128 2^-24 of the sum of their products' sizes, 2 * 128."""
    q, cache, table, lens, starts = _case([(new, 400), (1, 333), (min(new, 77), 77)], 6, 2, dim, dtype, cache_dtype, seed=60)
    out = serving.paged_attention(q, cache, table, lens, starts, max_new=new, scale=2.0)
    want, _, size = _attend64(q, cache, table, lens, starts, scale=2.0)
    tail = 400 * 2.0**-39 * 6 if dtype == "f16" or cache_dtype in TOP else 0.0
    off = (out.double() - want).abs() - (U[q.dtype] * (want.abs() + size) + 128 * 2.0**-24 * 256 * size + tail + (2.0**-25 if dtype == "f16" else 0))
    assert (off <= 0).all(), off.max().item()
