"""The serving operators together in a decoder, and what their kernels do when a wait runs out."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT / "examples"))

from paged_decoder import Config, PagedDecoder, mlp_plan, projection_plan  # noqa: E402

from mlir_gpu_kernel_compiler_b200 import runtime as rt  # noqa: E402
from mlir_gpu_kernel_compiler_b200 import serving, toolchain  # noqa: E402


def test_the_decoders_plans_make_kernels():
    from mlir_gpu_kernel_compiler_b200.codegen import generate
    from mlir_gpu_kernel_compiler_b200.fuse import fuse

    for plan, kernels in ((projection_plan(Config()), 2), (mlp_plan(Config()), 4)):
        assert len(plan.kernels) == kernels and len(list(generate(fuse(plan)))) == kernels


# Two layers of bf16 activations: each stage rounds to 2^-8 of its values, some dozen roundings whose
# errors add like independent ones; the framework's bound for bf16 programs is 2e-2 of the norm.  An i8 cache
# adds 1 / 254 of a row's largest element, an e4m3 one 2^-4 of every element of k and v, averaged over keys.
@pytest.mark.gpu
@pytest.mark.parametrize("cache,tol", [("bf16", 2e-2), ("i8", 3e-2), ("e4m3", 1e-1)])
def test_decoder_in_chunks_and_single_tokens_is_the_dense_decoder(cache, tol):
    model = PagedDecoder(Config(cache=cache))
    gen = torch.Generator().manual_seed(3)
    tokens = {s: torch.randint(0, 512, (n,), generator=gen).tolist() for s, n in ((7, 150), (2, 17), (5, 33))}
    steps = [{7: tokens[7][:64]}, {7: tokens[7][64:90], 2: tokens[2][:16], 5: tokens[5][:1]}, {5: tokens[5][1:32], 7: tokens[7][90:120]},
             {7: tokens[7][120:149]}, {7: tokens[7][149:], 2: tokens[2][16:], 5: tokens[5][32:]}]
    at = dict.fromkeys(tokens, 0)
    want = {s: model.dense_logits(t) for s, t in tokens.items()}
    for new in steps:
        got = model.step(new)
        for i, (s, ts) in enumerate(new.items()):
            at[s] += len(ts)
            ref = want[s][at[s] - 1]
            assert (got[i] - ref).norm() <= tol * ref.norm(), (s, at[s])
    serving.check()
    assert at == {s: len(t) for s, t in tokens.items()}
    for s in tokens:
        model.finish(s)
    assert sorted(model.free) == list(range(model.config.pages))


@pytest.mark.gpu
def test_decoder_generates_the_same_whatever_pages_a_sequence_gets():
    model = PagedDecoder()
    prompts = [[5, 9, 2], list(range(100)), [1] * 65]
    first = model.generate(prompts, 6)
    assert model.generate(prompts, 6) == first and all(len(t) == 6 for t in first)
    with pytest.raises(ValueError, match="at most 64"):
        model.step({0: [1] * 65})


@pytest.mark.gpu
def test_8_bit_rows_on_8_bytes_are_written_and_read_but_not_attended():
    def pool():
        return torch.zeros(4, 16, 2, 72, dtype=torch.int8, device="cuda")[..., :64]

    scales = [torch.zeros(4, 16, 2, device="cuda") for _ in range(2)]
    odd, plain = serving.PagedCache(pool(), pool(), *scales), serving.PagedCache.empty(4, 16, 2, 64, "i8")
    x, slots = torch.randn(40, 2, 64, device="cuda"), torch.arange(40, device="cuda", dtype=torch.int32)
    for cache in (odd, plain):
        serving.cache_write(cache, x, -x, slots)
    assert torch.equal(odd.k, plain.k) and torch.equal(odd.v, plain.v)
    for a, b in zip(serving.cache_read(odd, slots), serving.cache_read(plain, slots)):
        assert torch.equal(a, b)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    one = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    with pytest.raises((ValueError, rt.RuntimeError_), match="16-byte"):
        serving.paged_attention(q, odd, one, one[0] + 1)
    serving.check()


_STALL_CHILD = textwrap.dedent("""
    import ctypes, sys
    import torch
    sys.path.insert(0, sys.argv[2])
    from mlir_gpu_kernel_compiler_b200 import runtime as rt
    rt._lib = lib = rt.library(sys.argv[1])            # the failure-path test build of the library
    from mlir_gpu_kernel_compiler_b200 import serving
    serving._native.init(sys.argv[1], rt.RuntimeError_, torch.OutOfMemoryError)
    for dtype in ("bf16", "i8"):
        cache = serving.PagedCache.empty(256, 16, 8, 128, dtype)
        table = torch.arange(256, device="cuda", dtype=torch.int32)[None]
        lens, starts = torch.tensor([4096], device="cuda"), torch.tensor([0, 512], device="cuda")
        q = torch.zeros(512, 32, 128, dtype=torch.bfloat16, device="cuda")
        serving.paged_attention(q, cache, table, lens, starts, max_new=512)
        try:
            serving.check()
        except rt.RuntimeError_ as e:
            print("RESULT", e)
        serving.check()                                  # the read cleared it; the context is usable
    y = serving.cache_read(cache, table[0])
    serving.check()
    print("AFTER", bool((y[0] == 0).all()))
""")


@pytest.mark.gpu
def test_a_wait_of_the_attention_kernel_that_runs_out_is_reported():
    """A test build whose producers never bring the first keys, with the wait limit lowered to 20 ms: the call
    returns, ``check`` names the wait, and the device goes on.  In a child process, away from the
    product library."""
    lib = toolchain.build_runtime(extra_flags=toolchain.STALL_TEST_FLAGS, variant="stalltest")
    r = subprocess.run([sys.executable, "-c", _STALL_CHILD, str(lib), str(ROOT)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [x for x in r.stdout.splitlines() if x.startswith("RESULT")]
    assert len(lines) == 2 and all("paged_attention: wait timeout" in x for x in lines), r.stdout
    assert "AFTER True" in r.stdout


@pytest.mark.gpu
def test_a_refused_step_changes_nothing():
    model = PagedDecoder(Config(pages=6, positions=90))
    tokens = list(range(60))
    model.step({0: tokens[:20]})
    state = list(model.free), {s: list(p) for s, p in model.pages.items()}, dict(model.lengths)
    for new, why, what in (({1: [1] * 65}, ValueError, "at most 64"), ({0: [1] * 50, 1: [2] * 20}, ValueError, "at most 64"), ({0: [1] * 71}, ValueError, "positions"),
                           ({1: [1] * 60, 0: [2] * 4, 2: []}, ValueError, "no new token"), ({}, ValueError, "at least 1"), ({1: [1] * 33, 2: [2] * 17}, RuntimeError, "no free page")):
        with pytest.raises(why, match=what):
            model.step(new)
        assert state == (list(model.free), model.pages, model.lengths)
    got = model.step({0: tokens[20:60]})[0]
    want = model.dense_logits(tokens)[-1]
    assert (got - want).norm() <= 2e-2 * want.norm()
    serving.check()


@pytest.mark.gpu
@pytest.mark.parametrize("cache,tol", [("bf16", 2e-2), ("i8", 3e-2), ("e4m3", 1e-1)])
def test_decoder_in_long_chunks_reaches_the_kernel_of_many_rows(cache, tol):
    """The same bounds as for short chunks; which kernel a chunk gets is told by the workspace that it asks for."""
    import ctypes
    import struct

    from paged_decoder import LONG_CHUNKS

    model = PagedDecoder(Config(cache=cache, **LONG_CHUNKS))
    c = model.config
    size, count, pool = ctypes.c_int64(), ctypes.c_int64(), model.caches[0]
    args = struct.pack("=21qd2q", 16, 16, 0, 16, 16, 16, 0, 0, c.rows, 1, c.q_heads, c.rows, 64, 64, c.q_heads * 128, 128, c.q_heads * 128, 128, 2, 1, 0,
                       0.1, 0, 0) + pool._native[:15 * 8]
    assert rt.library().tj_b200_paged_attention_workspace(args, ctypes.byref(size), ctypes.byref(count)) == rt.TJ_OK
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert size.value == 2 * sms * 256 * (128 * 4 + 8)  # two parts of 256 rows a multiprocessor
    gen = torch.Generator().manual_seed(4)
    tokens = {s: torch.randint(0, 512, (n,), generator=gen).tolist() for s, n in ((0, 1013), (1, 140))}
    want = {s: model.dense_logits(t) for s, t in tokens.items()}
    at = dict.fromkeys(tokens, 0)
    for new in ({0: 512}, {0: 372, 1: 140}, {0: 128}, {0: 1}):
        got = model.step({s: tokens[s][at[s]:at[s] + n] for s, n in new.items()})
        for i, (s, n) in enumerate(new.items()):
            at[s] += n
            assert (got[i] - want[s][at[s] - 1]).norm() <= tol * want[s][at[s] - 1].norm(), (s, at[s])
    serving.check()
    assert at == {s: len(t) for s, t in tokens.items()}
