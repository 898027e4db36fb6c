"""A small decoder that serves several sequences from one paged cache.

The dense parts of a layer are two compiled programs (``B200Program``: normalisation and the fused
projection; output projection, normalisation and the MLP); between them ``serving.rotary_cache_write`` turns
queries and keys and puts keys and values into the cache, and ``serving.paged_attention`` reads it.  A step
takes any mix of new tokens: chunks of prompts and single tokens of running sequences.

    python examples/paged_decoder.py            # three prompts in chunks, then greedy tokens for all
"""
from __future__ import annotations

import sys
from dataclasses import dataclass
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from mlir_gpu_kernel_compiler_b200 import B200Program, serving  # noqa: E402
from mlir_gpu_kernel_compiler_b200.plan import PProgram  # noqa: E402


@dataclass
class Config:
    layers: int = 2
    width: int = 256
    q_heads: int = 4
    kv_heads: int = 2
    head_dim: int = 64
    hidden: int = 512
    vocab: int = 512
    positions: int = 1024
    rows: int = 64            # rows of the compiled programs: the most tokens of one step
    pages: int = 64
    page_size: int = 16
    cache: str = "bf16"


# chunks of 512 tokens, which attention takes with its kernel of many rows
LONG_CHUNKS = dict(width=512, q_heads=8, kv_heads=2, head_dim=128, hidden=1024, rows=512, pages=128)


class _Plan:
    """A plan of row normalisations and GEMMs in tensorjit's JSON form."""

    def __init__(self, name):
        self.d = dict(format="tensorjit-plan/1", name=name, nodes=[], inputs=[], outputs=[], kernels=[], aliases={}, meta={})

    def node(self, op, inputs, shape, **attrs):
        i = len(self.d["nodes"])
        self.d["nodes"].append(dict(id=i, op=op, name=f"%{op}{i}", inputs=list(inputs), shape=list(shape), dtype="bf16", attrs=attrs))
        if op == "input":
            self.d["inputs"].append(i)
        return i

    def shape(self, i):
        return self.d["nodes"][i]["shape"]

    def kernel(self, kind, nodes, inputs, outputs, shape, anchor=None, **more):
        return dict(kind=kind, nodes=nodes, anchor=anchor, inputs=inputs, outputs=outputs, iter_shape=list(shape), **more)

    def norm(self, x, g):
        """(x - mean) / sqrt(var + 1e-5) * g"""
        shape = self.shape(x)
        one = [shape[0], 1]
        mean = self.node("mean", [x], one, axis=-1, keepdim=True)
        d = self.node("sub", [x, mean], shape)
        sq = self.node("mul", [d, d], shape)
        var = self.node("mean", [sq], one, axis=-1, keepdim=True)
        eps = self.node("const", [], [], value=1e-5)
        add = self.node("add", [var, eps], one)
        r = self.node("rsqrt", [add], one)
        n = self.node("mul", [d, r], shape)
        y = self.node("mul", [n, g], shape)
        k = self.kernel
        stages = [k("reduce", [mean], [x], [mean], shape, mean), k("elementwise", [d, sq], [x, mean], [d, sq], shape),
                  k("reduce", [var, add, r], [sq], [r], shape, var), k("elementwise", [n, y], [d, r, g], [y], shape)]
        self.d["kernels"].append(k("row", [mean, d, sq, var, add, r, n, y], [x, g], [y], shape, stages=stages,
                                   rows=[shape[0]], n=shape[1]))
        return y

    def linear(self, x, w, bias=None, gelu=False, residual=None):
        """x w^T (+ bias) (gelu) (+ residual), one kernel"""
        shape = [self.shape(x)[0], self.shape(w)[0]]
        m = y = self.node("matmul", [x, w], shape, trans_b=True)
        nodes, ins = [m], [x, w]
        if bias is not None:
            y = self.node("add", [y, bias], shape)
            nodes.append(y)
            ins.append(bias)
        if gelu:
            y = self.node("gelu", [y], shape)
            nodes.append(y)
        if residual is not None:
            y = self.node("add", [residual, y], shape)
            nodes.append(y)
            ins.append(residual)
        self.d["kernels"].append(self.kernel("matmul", nodes, ins, [y], shape, m))
        return y

    def done(self, *outputs):
        self.d["outputs"] = list(outputs)
        return PProgram.from_dict(self.d)


def projection_plan(c: Config) -> PProgram:
    """(x, g, w_qkv) -> norm(x) w_qkv^T"""
    p = _Plan("decoder_projection")
    x = p.node("input", [], [c.rows, c.width])
    g = p.node("input", [], [c.width])
    w = p.node("input", [], [(c.q_heads + 2 * c.kv_heads) * c.head_dim, c.width])
    return p.done(p.linear(p.norm(x, g), w))


def mlp_plan(c: Config) -> PProgram:
    """(x, o, w_o, g, w_1, b_1, w_2, b_2) -> h + gelu(norm(h) w_1^T + b_1) w_2^T + b_2,  h = x + o w_o^T"""
    p = _Plan("decoder_mlp")
    x = p.node("input", [], [c.rows, c.width])
    o = p.node("input", [], [c.rows, c.q_heads * c.head_dim])
    wo = p.node("input", [], [c.width, c.q_heads * c.head_dim])
    g = p.node("input", [], [c.width])
    w1, b1 = p.node("input", [], [c.hidden, c.width]), p.node("input", [], [c.hidden])
    w2, b2 = p.node("input", [], [c.width, c.hidden]), p.node("input", [], [c.width])
    h = p.linear(o, wo, residual=x)
    return p.done(p.linear(p.linear(p.norm(h, g), w1, b1, gelu=True), w2, b2, residual=h))


class PagedDecoder:
    def __init__(self, config: Config = Config(), device="cuda", seed: int = 0):
        c = self.config = config
        self.device = torch.device(device)
        gen = torch.Generator().manual_seed(seed)

        def w(*shape, scale):
            return (torch.randn(shape, generator=gen) * scale).to(torch.bfloat16).to(self.device)

        qkv, inner = (c.q_heads + 2 * c.kv_heads) * c.head_dim, c.q_heads * c.head_dim
        self.embedding = w(c.vocab, c.width, scale=1.0)
        self.head = w(c.vocab, c.width, scale=c.width**-0.5)
        self.weights = [dict(g1=1 + w(c.width, scale=0.1), wqkv=w(qkv, c.width, scale=c.width**-0.5), wo=w(c.width, inner, scale=inner**-0.5),
                             g2=1 + w(c.width, scale=0.1), w1=w(c.hidden, c.width, scale=c.width**-0.5), b1=w(c.hidden, scale=0.1),
                             w2=w(c.width, c.hidden, scale=c.hidden**-0.5), b2=w(c.width, scale=0.1)) for _ in range(c.layers)]
        self.project = B200Program(projection_plan(c), device=self.device)
        self.mlp = B200Program(mlp_plan(c), device=self.device)
        self.table = serving.rotary_table(c.head_dim, c.positions, device=self.device)
        self.caches = [serving.PagedCache.empty(c.pages, c.page_size, c.kv_heads, c.head_dim, c.cache, self.device) for _ in range(c.layers)]
        self.free = list(range(c.pages))
        self.pages: dict[int, list[int]] = {}   # of each sequence, in order
        self.lengths: dict[int, int] = {}

    def step(self, new: dict[int, list[int]]) -> torch.Tensor:
        """New tokens of some sequences, ``{sequence: tokens}``: the logits after each one's last, f32 [len(new), vocab]."""
        c, size = self.config, self.config.page_size
        tokens, slots, positions, starts = [], [], [], [0]
        need = 0   # everything that can be refused is, before a page or a length changes
        for s, ts in new.items():
            if not ts:
                raise ValueError(f"sequence {s}: no new token")
            have = self.lengths.get(s, 0) + len(ts)
            if have > c.positions:
                raise ValueError(f"sequence {s}: more than {c.positions} positions")
            need += -(-have // size) - len(self.pages.get(s, ()))
        n = sum(len(ts) for ts in new.values())
        if not 0 < n <= c.rows:
            raise ValueError(f"{n} new tokens, at least 1 and at most {c.rows}")
        if need > len(self.free):
            raise RuntimeError("no free page")
        for s, ts in new.items():
            have, pages = self.lengths.get(s, 0), self.pages.setdefault(s, [])
            while len(pages) * size < have + len(ts):
                pages.append(self.free.pop())
            at = range(have, have + len(ts))
            tokens += ts
            positions += at
            slots += [pages[i // size] * size + i % size for i in at]
            starts.append(len(tokens))
            self.lengths[s] = have + len(ts)
        pad = c.rows - n   # rows of no sequence: their slot is -1, attention does not reach them
        width = max(len(self.pages[s]) for s in new)

        def ints(x):
            return torch.tensor(x, dtype=torch.int32, device=self.device)

        table = ints([self.pages[s] + [0] * (width - len(self.pages[s])) for s in new])
        lens, starts = ints([self.lengths[s] for s in new]), ints(starts)
        slots, positions = ints(slots + [-1] * pad), ints(positions + [0] * pad)
        x = self.embedding[ints(tokens + [0] * pad).long()]
        hq, hk, most = c.q_heads, c.kv_heads, max(len(t) for t in new.values())
        o = torch.zeros(c.rows, hq, c.head_dim, dtype=x.dtype, device=self.device)
        for w, cache in zip(self.weights, self.caches):
            qkv = self.project(x, w["g1"], w["wqkv"])[0].view(c.rows, hq + 2 * hk, c.head_dim)
            q = serving.rotary_cache_write(cache, qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], slots, positions, self.table)
            serving.paged_attention(q, cache, table, lens, starts, max_new=most, out=o)
            x = self.mlp(x, o.view(c.rows, -1), w["wo"], w["g2"], w["w1"], w["b1"], w["w2"], w["b2"])[0]
        return (x[starts[1:].long() - 1] @ self.head.T).float()

    def prefill(self, prompts: dict[int, list[int]]) -> torch.Tensor:
        """Prompts through the cache in chunks, one sequence after the other; logits after each one's last token."""
        rows = self.config.rows
        got = []
        for s, ts in prompts.items():
            for i in range(0, len(ts), rows):
                logits = self.step({s: ts[i:i + rows]})
            got.append(logits)
        return torch.cat(got)

    def finish(self, sequence: int) -> None:
        """Give a sequence's pages back."""
        self.free += self.pages.pop(sequence)
        del self.lengths[sequence]

    def generate(self, prompts: list[list[int]], count: int) -> list[list[int]]:
        """Greedy tokens after each prompt."""
        logits, out = self.prefill(dict(enumerate(prompts))), [[] for _ in prompts]
        for i in range(count):
            for s, t in enumerate(logits.argmax(-1).tolist()):
                out[s].append(t)
            if i + 1 < count:
                logits = self.step({s: [o[-1]] for s, o in enumerate(out)})
        for s in range(len(prompts)):
            self.finish(s)
        serving.check(self.device)
        return out

    def dense_logits(self, tokens: list[int]) -> torch.Tensor:
        """The same decoder in f32 over a whole sequence, without a cache: logits after every token."""
        c, n = self.config, len(tokens)
        d, half, group = c.head_dim, c.head_dim // 2, c.q_heads // c.kv_heads
        cos, sin = self.table[:n, None, :half], self.table[:n, None, half:]
        x = self.embedding[tokens].float()

        def norm(v, g):
            v = v - v.mean(-1, keepdim=True)
            return v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * g.float()

        def turn(v):
            a, b = v[..., :half], v[..., half:]
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        hidden = torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1)
        for w in self.weights:
            q, k, v = (norm(x, w["g1"]) @ w["wqkv"].float().T).view(n, -1, d).split([c.q_heads, c.kv_heads, c.kv_heads], 1)
            q, k, v = turn(q), turn(k).repeat_interleave(group, 1), v.repeat_interleave(group, 1)
            s = torch.einsum("qhd,khd->hqk", q, k) * d**-0.5
            o = torch.einsum("hqk,khd->qhd", s.masked_fill(hidden, -torch.inf).softmax(-1), v)
            h = x + o.reshape(n, -1) @ w["wo"].float().T
            y = torch.nn.functional.gelu(norm(h, w["g2"]) @ w["w1"].float().T + w["b1"].float())
            x = h + y @ w["w2"].float().T + w["b2"].float()
        return x @ self.head.float().T


def main() -> None:
    gen = torch.Generator().manual_seed(1)
    for cache in ("bf16", "i8", "e4m3"):
        model = PagedDecoder(Config(cache=cache))
        prompts = [torch.randint(0, 512, (n,), generator=gen).tolist() for n in (5, 100, 70)]
        got = model.prefill(dict(enumerate(prompts)))
        want = torch.stack([model.dense_logits(p)[-1] for p in prompts])
        print(f"{cache} cache: logits off by {((got - want).norm() / want.norm()).item():.4f} of their norm")
        for s in range(len(prompts)):
            model.finish(s)
        for p, t in zip(prompts, model.generate(prompts, 12)):
            print(f"  {len(p)} prompt tokens -> {t}")


if __name__ == "__main__":
    main()
