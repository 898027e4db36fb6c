"""Cases of the serving operators: rotary positions, the paged cache's writes and reads, attention over that cache.

``listed()`` and ``draw()`` give cases, ``prepare()`` a case's inputs on the GPU, ``run()`` one pass: in elementary
torch operations where ``own`` is false, through ``mlir_gpu_kernel_compiler_b200.serving`` where it is true.
``work()`` counts what a pass has to read, write and compute; ``exact()`` computes it in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i8": 1, "e4m3": 1}
TOP = {"i8": 127.0, "e4m3": 448.0}  # the largest code of a quantised cache


def listed():
    return [
        # one decoding step of 16 sequences: queries and keys of single tokens, where the launch is what costs
        dict(name="rotary_tokens", op="rotary", tokens=16, q_heads=32, kv_heads=8, dim=128, rot=128, layout="half", dtype="bf16",
             scaling="none", inverse=False),
        # a long prompt whose heads are rotated in their first half only, read out of the fused projection's rows
        dict(name="rotary_prompt", op="rotary", tokens=16384, q_heads=32, kv_heads=8, dim=128, rot=64, layout="interleaved",
             dtype="f16", scaling="ramp", inverse=False),
        # one decoding step of 64 sequences into an 8-bit cache: rotate, quantise, write, and the written tokens read back
        dict(name="append_tokens", op="append", tokens=64, q_heads=32, kv_heads=8, dim=128, rot=128, layout="half", dtype="bf16",
             cache="i8", page=16, order="token", scaling="linear"),
        # a prompt's tokens rotated and written to a 16-bit cache in one call
        dict(name="append_prompt", op="append", tokens=8192, q_heads=32, kv_heads=8, dim=128, rot=128, layout="half", dtype="bf16",
             cache="bf16", page=32, order="token", scaling="none"),
        # a chunk of an odd length quantised to 8-bit floats as it is written, and read back
        dict(name="cache_chunk", op="cache", tokens=509, read=509, kv_heads=8, dim=96, dtype="f16", cache="e4m3", page=16, order="head"),
        # a long context read back from an 8-bit cache after its last chunk was written
        dict(name="cache_long", op="cache", tokens=4096, read=32768, kv_heads=8, dim=128, dtype="bf16", cache="i8", page=64, order="token"),
        # one new token of one sequence with a head size of 64 and 16 heads: the smallest call
        dict(name="decode_one", op="attention", batch=1, new=1, context=777, q_heads=16, kv_heads=16, dim=64, dtype="bf16",
             cache="bf16", page=16, order="token", window=0, lse=False, ragged=False),
        # one decoding step of 64 sequences of uneven lengths, four query heads to a cached head
        dict(name="decode_batch", op="attention", batch=64, new=1, context=8192, q_heads=32, kv_heads=8, dim=128, dtype="bf16",
             cache="bf16", page=16, order="token", window=0, lse=False, ragged=True),
        # single tokens of three sequences over very long contexts in an 8-bit cache
        dict(name="decode_long", op="attention", batch=3, new=1, context=100003, q_heads=32, kv_heads=4, dim=128, dtype="bf16",
             cache="i8", page=64, order="head", window=0, lse=False, ragged=True),
        # a few new tokens a sequence (drafted tokens to be checked), a sliding window, seven query heads to a cached head
        dict(name="chunk_short", op="attention", batch=5, new=37, context=3001, q_heads=28, kv_heads=4, dim=64, dtype="f16",
             cache="e4m3", page=16, order="token", window=1024, lse=True, ragged=True),
        # a chunk of a long prompt over the cached rest of it: the largest
        dict(name="chunk_prompt", op="attention", batch=1, new=2048, context=16384, q_heads=32, kv_heads=8, dim=128, dtype="bf16",
             cache="bf16", page=32, order="token", window=0, lse=False, ragged=False),
        # prompts' chunks and single tokens of eight sequences in one call, over an 8-bit cache
        dict(name="chunk_mixed", op="attention", batch=8, new=1000, context=6000, q_heads=32, kv_heads=8, dim=128, dtype="bf16",
             cache="i8", page=16, order="token", window=0, lse=True, ragged=True),
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over their logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "cache", "attention", "attention", "attention"))
    kv = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 4, 5, 7, 8))
    scaling = rng.choice(("none", "linear", "ramp"))
    if op == "rotary":
        dim = rng.choice((64, 80, 96, 128, 256))
        return dict(op=op, tokens=_spread(rng, 1, 8192), q_heads=kv * min(group, 4), kv_heads=kv, dim=dim,
                    rot=rng.choice((dim, dim, dim // 2, 20)), layout=rng.choice(("half", "interleaved")),
                    dtype=rng.choice(("bf16", "f16", "f32")), scaling=scaling, inverse=rng.random() < 0.3)
    page = rng.choice((8, 16, 24, 32, 64, 128))
    order = rng.choice(("token", "head"))
    dtype = rng.choice(("bf16", "f16"))
    cache = rng.choice((dtype, "i8", "e4m3"))
    if op == "append":
        dim = rng.choice((64, 96, 128))
        return dict(op=op, tokens=_spread(rng, 1, 8000), q_heads=kv * min(group, 4), kv_heads=kv, dim=dim,
                    rot=rng.choice((dim, dim // 2)), layout=rng.choice(("half", "interleaved")), dtype=dtype, cache=cache, page=page,
                    order=order, scaling=scaling)
    if op == "cache":
        tokens = _spread(rng, 1, 4096)
        return dict(op=op, tokens=tokens, read=_spread(rng, 1, 30000), kv_heads=kv, dim=rng.choice((64, 80, 96, 128, 256)),
                    dtype=dtype, cache=rng.choice(("i8", "e4m3", dtype)), page=page, order=order)
    new = 1 if rng.random() < 0.4 else _spread(rng, 2, 2048)
    batch = _spread(rng, 1, max(1, min(64, 4096 // new)))
    most = min(100000 if cache != dtype else 50000, 600000 // batch)  # tokens of a sequence
    if new > 1:
        most = min(most, 960000000 // (new * batch * kv * group))  # the work of the largest listed case
    return dict(op=op, batch=batch, new=new, context=new + _spread(rng, 1, max(2, most)), q_heads=kv * group, kv_heads=kv,
                dim=rng.choice((64, 128)), dtype=dtype, cache=cache, page=page, order=order,
                window=rng.choice((0, 0, 0, 500)), lse=rng.random() < 0.5, ragged=rng.random() < 0.7)


# ---- what a case stands for ------------------------------------------------------------------------------------


def _lengths(case):
    """(new tokens, context) of each sequence of an attention case; the context counts the new tokens."""
    rng = random.Random(case["batch"] * 1000003 + case["context"] * 101 + case["new"])
    got = []
    for b in range(case["batch"]):
        new, context = case["new"], case["context"]
        if case["ragged"] and b:
            new = 1 if rng.random() < 0.3 else rng.randint(1, new)
            context = max(new, rng.randint(context // 3, context))
        got.append((new, context))
    return got


def _pairs(case):
    """(query token, visible key) pairs, and keys that some query sees, over all sequences."""
    pairs = keys = 0
    w = case["window"] or 1 << 40
    for n, c in _lengths(case):
        full = min(max(c - w, 0), n)  # the last `full` tokens see exactly w keys
        rest = n - full
        pairs += full * w + rest * (c - n) + rest * (rest + 1) // 2
        keys += min(c, w + n - 1)
    return pairs, keys


def work(case):
    d = case["dim"]
    if case["op"] == "rotary":
        rows = case["tokens"] * (case["q_heads"] + case["kv_heads"])
        return {"bytes": 2 * rows * d * SIZE[case["dtype"]] + case["tokens"] * (4 * case["rot"] + 4), "flops": 3 * rows * case["rot"]}
    e, c = SIZE[case["dtype"]], SIZE[case["cache"]]
    scale = 4 if case["cache"] in TOP else 0
    if case["op"] == "append":
        t, rows = case["tokens"], 2 * case["tokens"] * case["kv_heads"]
        turned = t * (case["q_heads"] + case["kv_heads"])
        b = 2 * t * case["q_heads"] * d * e + rows * (d * (e + c) + scale) + t * (4 * case["rot"] + 8)
        if scale:
            b += rows * (d * (c + e) + scale) + 4 * t
        return {"bytes": b, "flops": 3 * turned * case["rot"] + rows * d * (4 if scale else 0)}
    if case["op"] == "cache":
        w, r = 2 * case["tokens"] * case["kv_heads"], 2 * case["read"] * case["kv_heads"]
        return {"bytes": (w + r) * (d * (e + c) + scale) + 4 * (case["tokens"] + case["read"]), "flops": (3 * w + r) * d}
    pairs, keys = _pairs(case)
    tokens = sum(n for n, _ in _lengths(case))
    b = 2 * tokens * case["q_heads"] * d * e + 2 * keys * case["kv_heads"] * (d * c + scale) + 4 * keys // case["page"]
    return {"bytes": b + (4 * tokens * case["q_heads"] if case["lse"] else 0), "flops": 4 * d * pairs * case["q_heads"]}


# ---- inputs ----------------------------------------------------------------------------------------------------


def _table(case, positions):
    """cos and sin of the rotary angles, [positions, rot]: the cosines, then the sines."""
    half = case["rot"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    if case["scaling"] == "linear":  # positions drawn together by 4
        freq = freq / 4
    elif case["scaling"] == "ramp":  # slow frequencies drawn together by 8, fast ones kept, a ramp between
        turns = 4096 * freq / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        freq = freq * keep + freq / 8 * (1 - keep)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _pool(case, pages, gen):
    """An empty cache's four tensors: [pages, page, kv_heads, dim] for keys and values, in the order of tokens or of heads in
    memory, and for a quantised one the scales [pages, page, kv_heads]."""
    p, h, d = case["page"], case["kv_heads"], case["dim"]
    kind = DTYPES[case["cache"]]

    def some():
        if case["order"] == "token":
            return torch.zeros(pages, p, h, d, device="cuda", dtype=kind)
        return torch.zeros(pages, h, p, d, device="cuda", dtype=kind).transpose(1, 2)

    if case["cache"] not in TOP:
        return some(), some(), None, None
    return some(), some(), torch.zeros(pages, p, h, device="cuda"), torch.zeros(pages, p, h, device="cuda")


def _fill(t, gen):
    """Every slot of a cache's tensor holds some token's values, as in a pool that has been in use."""
    for part in t.split(max(1, (1 << 27) // max(1, t[0].numel()))):
        x = torch.randn(part.shape, device="cuda", generator=gen)
        part.copy_((x * 40).clamp(-127, 127).round() if t.dtype == torch.int8 else x * 60 if t.dtype == torch.float8_e4m3fn else x)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 7 + 1)
    kind = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen).to(kind)

    s = dict(case)
    if case["op"] == "rotary":
        t, hq, hk, d = case["tokens"], case["q_heads"], case["kv_heads"], case["dim"]
        rows = randn(t, hq + 2 * hk, d)  # the fused projection's output: queries, keys, values
        reach = max(2 * t, 4096)
        s.update(q=rows[:, :hq], k=rows[:, hq : hq + hk], table=_table(case, reach),
                 positions=torch.randint(0, reach, (t,), device="cuda", generator=gen).int())
        return s
    if case["op"] in ("append", "cache"):
        t, hk, d, page = case["tokens"], case["kv_heads"], case["dim"], case["page"]
        read = case.get("read", t)
        pages = -(-max(t, read) // page) + 3
        kc, vc, ks, vs = _pool(case, pages, gen)
        free = torch.randperm(pages * page, device="cuda", generator=gen)[: max(t, read)].int() if t <= 256 else (
            torch.randperm(pages, device="cuda", generator=gen)[:, None] * page + torch.arange(page, device="cuda")).reshape(-1)[: max(t, read)].int()
        for x in (kc, vc):
            _fill(x, gen)
        for x in (ks, vs):
            if x is not None:
                x.copy_(torch.rand(x.shape, device="cuda", generator=gen) * 0.02 + 0.01)
        s.update(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=free[-t:].clone(), read_slots=free[:read].clone())
        if case["op"] == "append":
            hq = case["q_heads"]
            rows = randn(t, hq + 2 * hk, d)
            s.update(q=rows[:, :hq], k=rows[:, hq : hq + hk], v=rows[:, hq + hk :], table=_table(case, max(2 * t, 4096)),
                     positions=torch.randint(0, max(2 * t, 4096), (t,), device="cuda", generator=gen).int())
        else:
            s.update(k=randn(t, hk, d), v=randn(t, hk, d))
        return s
    lens = _lengths(case)
    page = case["page"]
    wide = max(-(-c // page) for _, c in lens)
    need = sum(-(-c // page) for _, c in lens)
    order = torch.randperm(need + 5, device="cuda", generator=gen)[:need].int()
    table = torch.full((len(lens), wide), -1, device="cuda", dtype=torch.int32)
    at = 0
    for b, (_, c) in enumerate(lens):
        n = -(-c // page)
        table[b, :n] = order[at : at + n]
        at += n
    kc, vc, ks, vs = _pool(case, need + 5, gen)
    for x in (kc, vc):
        _fill(x, gen)
    for x in (ks, vs):
        if x is not None:
            x.copy_(torch.rand(x.shape, device="cuda", generator=gen) * 0.02 + 0.01)
    tokens = sum(n for n, _ in lens)
    starts = torch.tensor([0] + [n for n, _ in lens], device="cuda").cumsum(0).int()
    s.update(q=randn(tokens, case["q_heads"], case["dim"]), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=table,
             kv_lens=torch.tensor([c for _, c in lens], device="cuda", dtype=torch.int32), q_starts=starts)
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------


def _turn(x, s, inverse=False):
    """Rotary positions on [tokens, heads, dim], in 32 bits."""
    rot, half = s["rot"], s["rot"] // 2
    row = s["table"][s["positions"].long()][:, None]
    c, sn = row[..., :half], row[..., half:]
    if inverse:
        sn = -sn
    x = x.float()
    if s["layout"] == "half":
        a, b = x[..., :half], x[..., half:rot]
        turned = torch.cat((a * c - b * sn, b * c + a * sn), -1)
    else:
        a, b = x[..., :rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
    return torch.cat((turned, x[..., rot:]), -1)


def _put(cache, scale, x, slots, page):
    """Tokens' rows, in 32 bits, into the slots of one tensor of the cache."""
    at = (slots.long() // page, slots.long() % page)
    if scale is None:
        cache[at] = x.to(cache.dtype)
        return
    top = TOP["i8" if cache.dtype == torch.int8 else "e4m3"]
    s = x.abs().amax(-1) / top
    code = torch.where(s[..., None] > 0, x / s[..., None], 0.0)
    cache[at] = code.round().to(torch.int8) if cache.dtype == torch.int8 else code.to(cache.dtype)
    scale[at] = s


def _get(cache, scale, slots, page, kind):
    at = (slots.long() // page, slots.long() % page)
    x = cache[at].float()
    return (x if scale is None else x * scale[at][..., None]).to(kind)


def _attend(s):
    """Attention of the new tokens over their sequences' pages, padded to the longest of each."""
    b, hk, g, d, page = s["batch"], s["kv_heads"], s["q_heads"] // s["kv_heads"], s["dim"], s["page"]
    pages = s["page_table"].long().clamp(min=0)
    reach = pages.shape[1] * page
    at = torch.arange(reach, device="cuda")
    held = (at < s["kv_lens"][:, None])[..., None, None]  # what a page holds after its sequence's end is not read

    def dense(cache, scale):
        x = cache[pages].reshape(b, reach, hk, d).float()
        if scale is not None:
            x = x * scale[pages].reshape(b, reach, hk, 1)
        return torch.where(held, x, 0.0).transpose(1, 2)

    starts, new = s["q_starts"].long(), s["new"]
    i = torch.arange(new, device="cuda")
    count = starts[1:] - starts[:-1]
    token = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[token].reshape(b, new, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b, hk, g * new, d)
    score = (q @ dense(s["k_cache"], s["k_scale"]).transpose(2, 3)).view(b, hk, g, new, reach) * d**-0.5
    place = s["kv_lens"][:, None] - count[:, None] + i
    seen = (at <= place[..., None]) & (i < count[:, None])[..., None]
    if s["window"]:
        seen &= at > place[..., None] - s["window"]
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (score - top).exp()
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, hk, g * new, reach) @ dense(s["v_cache"], s["v_scale"])).view(b, hk, g, new, d) / torch.where(total > 0, total, 1.0)
    back = torch.repeat_interleave(torch.arange(b, device="cuda"), count, output_size=s["q"].shape[0])
    step = torch.arange(s["q"].shape[0], device="cuda") - starts[back]
    out = out.permute(0, 3, 1, 2, 4).reshape(b, new, hk * g, d)[back, step].to(s["q"].dtype)
    if not s["lse"]:
        return out
    return out, (top + total.log())[..., 0].permute(0, 3, 1, 2).reshape(b, new, hk * g)[back, step]


def _plain(s):
    if s["op"] == "rotary":
        return [_turn(x, s, s["inverse"]).to(x.dtype) for x in (s["q"], s["k"])]
    if s["op"] == "attention":
        return _attend(s)
    got = {}
    k, v = s["k"].float(), s["v"].float()
    if s["op"] == "append":
        got["q"] = _turn(s["q"], s).to(s["q"].dtype)
        k = _turn(s["k"], s)
    _put(s["k_cache"], s["k_scale"], k, s["slots"], s["page"])
    _put(s["v_cache"], s["v_scale"], v, s["slots"], s["page"])
    if s["op"] == "append" and s["k_scale"] is None:
        return got | {"k": s["k_cache"], "v": s["v_cache"]}
    kind = DTYPES[s["dtype"]]
    got["k"] = _get(s["k_cache"], s["k_scale"], s["read_slots"], s["page"], kind)
    got["v"] = _get(s["v_cache"], s["v_scale"], s["read_slots"], s["page"], kind)
    return got


def run(state):
    s = state
    if not own:
        return _plain(s)
    from mlir_gpu_kernel_compiler_b200 import serving

    if s["op"] == "rotary":
        return list(serving.rotary(s["q"], s["k"], s["positions"], s["table"], layout=s["layout"], inverse=s["inverse"]))
    cache = serving.PagedCache(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
    if s["op"] == "attention":
        return serving.paged_attention(s["q"], cache, s["page_table"], s["kv_lens"], s["q_starts"], max_new=s["new"],
                                       window=s["window"], return_lse=s["lse"])
    got = {}
    if s["op"] == "append":
        got["q"] = serving.rotary_cache_write(cache, s["q"], s["k"], s["v"], s["slots"], s["positions"], s["table"], layout=s["layout"])
        if s["k_scale"] is None:
            return got | {"k": s["k_cache"], "v": s["v_cache"]}
    else:
        serving.cache_write(cache, s["k"], s["v"], s["slots"])
    got["k"], got["v"] = serving.cache_read(cache, s["read_slots"], dtype=s["dtype"])
    return got


# ---- in 64 bits ------------------------------------------------------------------------------------------------


def _turn64(x, s, sign):
    """Each pair as a complex number times cos + i sin."""
    half, rot = s["rot"] // 2, s["rot"]
    x = x.double()
    row = s["table"].double()[s["positions"].long()]
    unit = torch.complex(row[:, :half], sign * row[:, half:])[:, None]
    y = x.clone()
    if s["layout"] == "half":
        z = torch.complex(x[..., :half], x[..., half:rot]) * unit
        y[..., :half], y[..., half:rot] = z.real, z.imag
    else:
        z = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * unit
        y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
    return y


def _code64(x, cache):
    """What a quantised cache holds of the rows x, as the values that it stands for."""
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.where(top > 0, top, 1.0) / TOP[cache]
    y = x / unit
    if cache == "i8":
        return y.round() * unit
    step = 2.0 ** (torch.where(y == 0, 1.0, y.abs()).log2().floor().clamp(min=-6) - 3)  # 3 bits after the leading one
    return (y / step).round() * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return [_turn64(x, s, -1 if case["inverse"] else 1) for x in (s["q"], s["k"])]
    if case["op"] != "attention":
        got, page, n = {}, s["page"], s["slots"].numel()
        new = [_turn64(s["k"], s, 1) if case["op"] == "append" else s["k"].double(), s["v"].double()]
        if case["op"] == "append":
            got["q"] = _turn64(s["q"], s, 1)
        where = torch.full((s["k_cache"].shape[0] * page,), -1, device="cuda")
        where[s["slots"].long()] = torch.arange(n, device="cuda")
        whole = case["op"] == "append" and case["cache"] not in TOP
        slots = torch.arange(where.numel(), device="cuda") if whole else s["read_slots"].long()
        for name, x in zip("kv", new):
            if case["cache"] in TOP:
                x = _code64(x, case["cache"])
            elif not whole:  # rounded as it is written, before it is read
                x = x.to(DTYPES[case["cache"]]).double()
            old = s[name + "_cache"][slots // page, slots % page].double()
            if s[name + "_scale"] is not None:
                old = old * s[name + "_scale"][slots // page, slots % page].double()[..., None]
            token = where[slots]
            y = torch.where((token >= 0)[:, None, None], x[token.clamp(min=0)], old)
            got[name] = y.reshape(s["k_cache"].shape) if whole else y
        return got
    lens = _lengths(case)
    g, d, page = case["q_heads"] // case["kv_heads"], case["dim"], case["page"]
    out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    lse = torch.full(s["q"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    at = 0
    for b, (n, c) in enumerate(lens):
        key = torch.arange(c, device="cuda")
        pg, sl = s["page_table"][b].long()[key // page], key % page
        place = torch.arange(c - n, c, device="cuda")
        hidden = key[None] > place[:, None]
        if case["window"]:
            hidden |= key[None] <= place[:, None] - case["window"]
        for h in range(case["kv_heads"]):
            k, v = s["k_cache"][pg, sl, h].double(), s["v_cache"][pg, sl, h].double()
            if s["k_scale"] is not None:
                k, v = k * s["k_scale"][pg, sl, h].double()[:, None], v * s["v_scale"][pg, sl, h].double()[:, None]
            for j in range(h * g, h * g + g):
                a = s["q"][at : at + n, j].double() @ k.T / math.sqrt(d)
                a.masked_fill_(hidden, -math.inf)
                lse[at : at + n, j] = a.logsumexp(1)
                out[at : at + n, j] = a.softmax(1) @ v
        at += n
    return (out, lse) if case["lse"] else out
