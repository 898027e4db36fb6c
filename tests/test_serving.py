"""The serving operators without a GPU: the layout of the C structures, and what is refused before a launch."""
import ctypes
import struct
import subprocess
from pathlib import Path

import pytest
import torch

from mlir_gpu_kernel_compiler_b200 import runtime as rt
from mlir_gpu_kernel_compiler_b200 import serving

HEADER = Path(__file__).resolve().parents[1] / "include" / "tj_b200.h"
# the C structures are 8-byte fields throughout
CACHE = struct.Struct("=15q")       # tj_kv_cache
ROWS = struct.Struct("=27q")        # tj_rows, without its cache
ATTENTION = struct.Struct("=21qd2q")  # tj_paged_attention, without its cache


def test_packed_structures_match_the_header(tmp_path):
    src = tmp_path / "sz.c"
    src.write_text(f'#include "{HEADER}"\n#include <stdio.h>\n#include <stddef.h>\n'
                   'int main(){printf("%zu %zu %zu %zu %zu %zu %zu\\n", sizeof(tj_kv_cache), offsetof(tj_rows, cache), '
                   "sizeof(tj_rows), offsetof(tj_rows, dtype), offsetof(tj_paged_attention, cache), "
                   "offsetof(tj_paged_attention, scale), sizeof(tj_paged_attention)); return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", str(src), "-o", str(exe)], check=True)
    vals = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    c, r, a = CACHE.size, ROWS.size, ATTENTION.size
    assert vals == [c, r, r + c, 24 * 8, a, 21 * 8, a + c]


def _cache(dtype=4, k=4096, v=8192, ks=4096, vs=4096, pages=4, page=16, heads=2, dim=64, strides=(2048, 128, 64), scale=(32, 2, 1)):
    return CACHE.pack(k, v, ks, vs, pages, page, heads, dim, *strides, *scale, dtype)


def _rows(q=0, k=4096, v=4096, q2=0, k2=0, slots=4096, pos=0, table=0, tokens=3, hq=0, hk=2, dim=64, rot=0, rows=0, stride=128, dtype=2):
    return ROWS.pack(q, k, v, q2, k2, slots, pos, table, tokens, hq, hk, dim, rot, rows, *[stride, 64] * 5, dtype, 0, 0)


BAD_CACHES = [(dict(k=0), b"NULL"), (dict(dtype=9), b"dtype"), (dict(ks=0), b"scales"), (dict(dtype=2), b"scales"), (dict(pages=0), b"positive"),
              (dict(pages=1 << 28), b"2\\^31"), (dict(dim=60), b"multiple of 8"), (dict(dim=520), b"multiple of 8"),
              (dict(strides=(2048, 130, 64)), b"boundaries"), (dict(k=4104), b"boundaries")]


@pytest.mark.parametrize("how,why", BAD_CACHES)
def test_c_entries_refuse_bad_caches(how, why):
    import re

    lib = rt.library()
    for rc in (lib.tj_b200_cache_write(_rows() + _cache(**how), None),
               lib.tj_b200_cache_read(_cache(**how), 4096, 3, 4096, 4096, 2, None)):
        assert rc == rt.TJ_ERR_INVALID and re.search(why, lib.tj_b200_last_error())


def test_c_entries_refuse_bad_rows():
    lib = rt.library()
    none = bytes(CACHE.size)
    for args, why in [(_rows(dtype=3) + _cache(), b"f32, f16 or bf16"), (_rows(dim=72) + _cache(), b"cache's heads"),
                      (_rows(hk=3) + _cache(), b"cache's heads"), (_rows(slots=0) + _cache(), b"slots"), (_rows(k=4100) + _cache(), b"boundaries"),
                      (_rows(stride=130) + _cache(), b"boundaries"), (_rows(rot=3) + _cache(), b"even"), (_rows(rot=66) + _cache(), b"even"),
                      (_rows(rot=64) + _cache(), b"positions"), (_rows(q=4096, hq=1) + _cache(), b"q needs an output"),
                      (_rows(tokens=-1) + _cache(), b"negative")]:
        assert lib.tj_b200_cache_write(args, None) == rt.TJ_ERR_INVALID and why in lib.tj_b200_last_error(), why
    for args, why in [(_rows(k=0, v=0, slots=0, rot=8, pos=16, table=16, rows=4), b"nothing"),
                      (_rows(v=0, slots=0, rot=8, pos=16, table=16, rows=4), b"k needs an output"),
                      (_rows(q=16, q2=16, rot=8, pos=16, table=16, rows=4), b"neither v nor slots"),
                      (_rows(q=16, q2=16, k=0, v=0, slots=0), b"rot must be positive")]:
        assert lib.tj_b200_rotary(args + none, None) == rt.TJ_ERR_INVALID and why in lib.tj_b200_last_error(), why
    assert lib.tj_b200_rotary(None, None) == lib.tj_b200_cache_write(None, None) == rt.TJ_ERR_INVALID
    assert lib.tj_b200_cache_read(None, None, 0, None, None, 0, None) == rt.TJ_ERR_INVALID
    assert lib.tj_b200_cache_read(_cache(), None, 3, None, None, 2, None) == rt.TJ_ERR_INVALID
    assert lib.tj_b200_cache_read(_cache(), 4096, 3, 4096, 4096, 3, None) == rt.TJ_ERR_INVALID
    assert lib.tj_b200_serving_status(None, None, None) == rt.TJ_ERR_INVALID


def test_c_entry_refuses_bad_attention():
    lib = rt.library()

    def args(q=4096, out=4096, starts=4096, tokens=5, batch=2, heads=4, max_new=3, width=4, dtype=2, window=0, scale=0.125, stride=256, ws=4096, cache=None):
        return ATTENTION.pack(q, out, 0, 4096, 4096, starts, ws, 4096, tokens, batch, heads, max_new, width, width, stride, 64, stride, 64,
                                       dtype, 1, window, scale, 1 << 40, 1 << 30) + (cache or _cache())

    for how, why in [(dict(dtype=0), b"f16 or bf16"), (dict(cache=_cache(dtype=1, ks=0, vs=0)), b"q's type"),
                     (dict(cache=_cache(dim=96)), b"64 or 128"), (dict(heads=3), b"multiple"), (dict(heads=0), b"extent"),
                     (dict(max_new=0), b"extent"), (dict(width=0), b"extent"), (dict(window=-1), b"extent"), (dict(tokens=-1), b"extent"),
                     (dict(starts=0), b"one token"), (dict(scale=0.0), b"scale"), (dict(scale=float("nan")), b"scale"),
                     (dict(cache=_cache(k=0)), b"NULL"), (dict(tokens=1 << 30), b"too many")]:
        assert lib.tj_b200_paged_attention(args(**how), None) == rt.TJ_ERR_INVALID and why in lib.tj_b200_last_error(), why
        size, count = ctypes.c_int64(), ctypes.c_int64()
        assert lib.tj_b200_paged_attention_workspace(args(**how), ctypes.byref(size), ctypes.byref(count)) == rt.TJ_ERR_INVALID
    for how, why in [(dict(q=0), b"NULL"), (dict(ws=0), b"NULL"), (dict(q=4100), b"boundaries"), (dict(stride=260), b"boundaries")]:
        assert lib.tj_b200_paged_attention(args(**how), None) == rt.TJ_ERR_INVALID and why in lib.tj_b200_last_error(), why
    assert lib.tj_b200_paged_attention(None, None) == rt.TJ_ERR_INVALID


def test_python_refusals_on_the_host():
    x = torch.zeros(2, 2, 64)
    with pytest.raises(TypeError, match="q: expected a torch.Tensor"):
        serving.rotary([1.0], None, x, x)
    with pytest.raises(ValueError, match="on cpu"):
        serving.rotary(x, None, torch.zeros(2), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="3 dimensions"):
        serving.rotary(x[0], None, torch.zeros(2), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="dtype"):
        serving.rotary(x.double(), None, torch.zeros(2), torch.zeros(4, 64))
    with pytest.raises(ValueError, match="on cpu"):
        serving.PagedCache(torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16), torch.zeros(2, 4, 2, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="dtype must be"):
        serving.PagedCache.empty(1, 1, 1, 64, dtype="f32")
    for call in (lambda: serving.cache_write(None, x, x, x), lambda: serving.cache_read(None, x), lambda: serving.paged_attention(x, None, x, x)):
        with pytest.raises(TypeError, match="PagedCache"):
            call()
    for how in (dict(rot_dim=3), dict(rot_dim=0), dict(max_positions=0), dict(scaling="other"), dict(factor=0.0), dict(scaling="ramp"),
                dict(scaling="ramp", original=8, fast=1.0), dict(scaling="base", rot_dim=2)):
        with pytest.raises(ValueError):
            serving.rotary_table(**{"rot_dim": 8, "max_positions": 4, "device": "cpu", **how})
    assert serving.rotary_table(8, 4, device="cpu").shape == (4, 8)


@pytest.mark.parametrize("strides", [(2048, 128, 72), (2048, 136, 64), (2056, 128, 64)])
def test_attention_refuses_cache_rows_that_only_start_on_8_bytes(strides):
    """The row operators take 8-bit rows at multiples of 8 bytes; attention copies 16 bytes at a time."""
    lib, size, count = rt.library(), ctypes.c_int64(), ctypes.c_int64()
    args = ATTENTION.pack(4096, 4096, 0, 4096, 4096, 4096, 4096, 4096, 5, 2, 4, 3, 4, 4, 256, 64, 256, 64, 2, 1, 0, 0.125,
                          1 << 40, 1 << 30) + _cache(strides=strides)
    assert lib.tj_b200_paged_attention(args, None) == rt.TJ_ERR_INVALID and b"16-byte" in lib.tj_b200_last_error()
    assert lib.tj_b200_paged_attention_workspace(args, ctypes.byref(size), ctypes.byref(count)) == rt.TJ_ERR_INVALID


def test_c_entry_refuses_bad_index_arrays():
    lib = rt.library()
    for args, why in [((4096, -1, 4, 4, 1, 4096), b"negative"), ((4096, 4, -1, 4, 1, 4096), b"negative"), ((0, 2, 2, 2, 1, 4096), b"NULL"),
                      ((4096, 2, 2, 2, 1, 0), b"NULL"), ((4096, 1 << 40, 1 << 20, 2, 1, 4096), b"too many")]:
        assert lib.tj_b200_narrow_indices(*args, None) == rt.TJ_ERR_INVALID and why in lib.tj_b200_last_error(), why
    assert lib.tj_b200_narrow_indices(None, 0, 3, 3, 1, None, None) == rt.TJ_OK


def test_a_built_tree_is_not_built_again_where_it_is_copied_to(tmp_path):
    import shutil
    import sys

    from mlir_gpu_kernel_compiler_b200 import toolchain

    toolchain.build_runtime(), toolchain.build_serving_module()
    root = Path(__file__).resolve().parents[1]
    shutil.copytree(root / "mlir_gpu_kernel_compiler_b200", tmp_path / "mlir_gpu_kernel_compiler_b200", ignore=shutil.ignore_patterns("obj", "*.o"))
    shutil.copytree(root / "include", tmp_path / "include")
    code = ("import subprocess\nfrom mlir_gpu_kernel_compiler_b200 import toolchain\nrun = subprocess.run\n"
            "def no_compiler(cmd, **how):\n    assert '-c' not in cmd and '-shared' not in cmd, cmd\n    return run(cmd, **how)\n"
            "subprocess.run = no_compiler\nprint(toolchain.build_runtime(), toolchain.build_serving_module())")
    r = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True)
    assert r.returncode == 0 and str(tmp_path) in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale"])
def test_a_caches_tensors_cannot_be_replaced(name):
    """The operators go by the memory that the cache was made with."""
    cache = object.__new__(serving.PagedCache)
    with pytest.raises(AttributeError):
        setattr(cache, name, torch.zeros(1))
