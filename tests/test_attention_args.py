"""What the attention and cache entry points refuse, before anything reaches a GPU (CPU only): the wrappers by exceptions,
the C-ABI by the library's "check failed" message."""
import os
import subprocess
import sys

import pytest
import torch

from qengine_amd import ops
from test_abi import LIB, ROOT

BF, F16, I32 = torch.bfloat16, torch.float16, torch.int32


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def cache(**kw):
    a = dict(layers=2, pages=8, page=16, kv_heads=2, d=64, slots=3, max_tokens=64, device="cpu")
    a.update(kw)
    return ops.KVCache.empty(**a)


PROMPT = [
    (dict(q=z(4, 4, 64, dtype=torch.float32)), TypeError),
    (dict(q=z(4, 4, 64, dtype=F16)), TypeError),                       # k and v of another type
    (dict(q=z(4, 3, 64)), ValueError),                                # 3 heads over 2
    (dict(q=z(4, 0, 64)), ValueError),
    (dict(q=z(5, 4, 64)), ValueError),                                # other rows than k's
    (dict(q=z(4, 4, 96), k=z(4, 2, 96), v=z(4, 2, 96)), ValueError),  # head size
    (dict(v=z(4, 1, 64)), ValueError),
    (dict(q=z(4, 4, 65)[:, :, 1:]), ValueError),                      # strides
    (dict(q=z(4, 4, 128)[:, :, ::2]), ValueError),
    (dict(q=z(4 * 4 * 64 + 1)[1:].view(4, 4, 64)), ValueError),       # alignment
    (dict(q=z(4, 256)), ValueError),
    (dict(cu=z(2, dtype=torch.int64)), TypeError),
    (dict(cu=z(0, dtype=I32)), ValueError),
    (dict(cu=z(4, dtype=I32)[::2]), ValueError),
    (dict(cu=z(4098, dtype=I32)), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=-1.0), ValueError),
    (dict(scale=float("nan")), ValueError),
    (dict(out=z(4, 4, 64, dtype=F16)), TypeError),
    (dict(out=z(4, 2, 64)), ValueError),
    (dict(), ValueError),                                             # all well, but not on a GPU
]


@pytest.mark.parametrize("change,error", PROMPT)
def test_prompt_refusals(change, error):
    a = dict(q=z(4, 4, 64), k=z(4, 2, 64), v=z(4, 2, 64), cu=torch.tensor([0, 4], dtype=I32))
    a.update(change)
    with pytest.raises(error):
        ops.attn_prompt(**a)


@pytest.mark.parametrize("change", [dict(d=96), dict(page=8), dict(page=48), dict(page=2048), dict(kv_heads=1025), dict(pages=0),
                                    dict(max_tokens=2 ** 31)])
def test_cache_refusals(change):
    with pytest.raises(ValueError):
        cache(**change)


def test_cache_types_and_strides():
    c = cache()
    for name, bad, error in [("k", c.k.float(), TypeError), ("v", c.v.half(), TypeError), ("v", c.v[:, :4], ValueError),
                             ("table", c.table.long(), TypeError), ("length", c.length[:2], ValueError), ("ref", c.ref[:4], ValueError),
                             ("held", c.held.long(), TypeError), ("k", c.k.transpose(2, 3).contiguous().transpose(2, 3), ValueError)]:
        a = dict(k=c.k, v=c.v, table=c.table, length=c.length, held=c.held, ref=c.ref)
        a[name] = bad
        with pytest.raises(error):
            ops.KVCache(**a)


def i32(*v):
    return torch.tensor(v, dtype=I32)


CALLS = [
    (lambda c: c.attend(2, z(1, 4, 64), i32(0), i32(0, 1), 1), ValueError),          # layer
    (lambda c: c.attend(0, z(1, 3, 64), i32(0), i32(0, 1), 1), ValueError),          # heads
    (lambda c: c.attend(0, z(1, 4, 128), i32(0), i32(0, 1), 1), ValueError),
    (lambda c: c.attend(0, z(1, 4, 64, dtype=F16), i32(0), i32(0, 1), 1), TypeError),
    (lambda c: c.attend(0, z(1, 4, 64), i32(0), i32(0, 1), 0), ValueError),
    (lambda c: c.attend(0, z(1, 4, 64), i32(0), i32(0, 1), 65), ValueError),
    (lambda c: c.attend(0, z(1, 4, 64), i32(0, 1), i32(0, 1), 1), ValueError),       # seqs against cu
    (lambda c: c.attend(0, z(1, 4, 64), i32(0).long(), i32(0, 1), 1), TypeError),
    (lambda c: c.attend(0, z(2, 4, 64), i32(0), i32(0, 1), 1, mask=z(1, dtype=torch.int64)), ValueError),
    (lambda c: c.attend(0, z(2, 4, 64), i32(0), i32(0, 1), 1, mask=z(2, dtype=I32)), TypeError),
    (lambda c: c.attend(0, z(1, 4, 64), i32(0), i32(0, 1), 1, scale=-0.1), ValueError),
    (lambda c: c.attend(0, z(1, 4, 64), z(4097, dtype=I32), z(4098, dtype=I32), 1), ValueError),
    (lambda c: c.attend(0, z(1, 4, 64), i32(0), i32(0, 1), 1), ValueError),          # not on a GPU
    (lambda c: c.append(0, z(2, 2, 64), z(2, 1, 64), i32(0), i32(0, 2)), ValueError),
    (lambda c: c.append(None, z(1, 2, 2, 64), z(1, 2, 2, 64), i32(0), i32(0, 2)), ValueError),
    (lambda c: c.append(-1, z(2, 2, 64), z(2, 2, 64), i32(0), i32(0, 2)), ValueError),
    (lambda c: c.append(0, z(2, 2, 64), z(2, 2, 64), i32(0, 1), i32(0, 2)), ValueError),
    (lambda c: c.append(0, z(2, 2, 64), z(2, 2, 64), i32(0), i32(0, 2)), ValueError),
    (lambda c: c.reserve(i32(0, 1), i32(1)), ValueError),
    (lambda c: c.reserve(z(1025, dtype=I32), z(1025, dtype=I32)), ValueError),
    (lambda c: c.fork(i32(0), i32(1).long()), TypeError),
    (lambda c: c.fork(z(1025, dtype=I32), z(1025, dtype=I32)), ValueError),
    (lambda c: c.release(i32(0).view(1, 1)), ValueError),
    (lambda c: c.release(i32(0), i32(0, 1)), ValueError),
    (lambda c: c.release(z(1025, dtype=I32)), ValueError),
    (lambda c: c.accept(i32(0), i32(1), path=z(1, 65, dtype=I32)), ValueError),
    (lambda c: c.accept(i32(0), i32(1), path=z(2, 4, dtype=I32)), ValueError),
    (lambda c: c.accept(i32(0), i32(1), length=i32(0)), ValueError),
    (lambda c: c.accept(i32(0), i32(1)), ValueError),
]


@pytest.mark.parametrize("call,error", CALLS)
def test_call_refusals(call, error):
    with pytest.raises(error):
        call(cache())


HEAD = f"""
import ctypes, sys
sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, "tests")!r}]
import torch
from qengine_amd import ops, attention
from qengine_amd.qe import typed
c = ops.KVCache.empty(2, 8, 16, 2, 64, 3, 64, device="cpu")
p = ctypes.addressof(c._c)
f = lambda name, sig, *a: typed(name, sig)(*a)
"""


@pytest.mark.parametrize("code,msg", [
    ("f('qe_kv_reserve', 'pppippp', p, 0, 0, 1025, 0, 16, 0)", "qe_kv_reserve: n = 1025"),
    ("f('qe_kv_fork', 'pppipp', p, 0, 0, -1, 0, 0)", "qe_kv_fork: n = -1"),
    ("f('qe_kv_fork', 'pppipp', p, 0, 0, 1, 0, 0)", "qe_kv_fork: null pointer"),
    ("f('qe_kv_release', 'pppip', 0, 0, 0, 1, 0)", "qe_kv_release: no cache"),
    ("c._c.page = 24; f('qe_kv_release', 'pppip', p, 0, 0, 1, 0)", "page 24"),
    ("c._c.d = 80; f('qe_kv_release', 'pppip', p, 0, 0, 1, 0)", "d 80"),
    ("c._c.width = 1 << 27; f('qe_kv_release', 'pppip', p, 0, 0, 1, 0)", "pass 2^30 tokens"),
    ("c._c.pages = 1 << 30; f('qe_kv_release', 'pppip', p, 0, 0, 1, 0)", "1073741824 pages"),
    ("c._c.token_stride = 1 << 24; f('qe_kv_release', 'pppip', p, 0, 0, 1, 0)", "16777216 elements apart"),
    ("c._c.token_stride = 4; f('qe_kv_release', 'pppip', p, 0, 0, 1, 0)", "strides must be multiples of 8"),
    ("f('qe_kv_append', 'piipppppiip', p, 1, 2, 0, 0, 0, 0, 0, 1, 1, 0)", "qe_kv_append: layers 1 .. 3 of 2"),
    ("f('qe_kv_accept', 'ppppiipp', p, 16, 16, 16, 65, 1, 0, 0)", "paths of 65"),
    ("f('qe_attn_tree', 'pipllpllpppiiipifp', p, 0, 16, 8, 8, 16, 8, 8, 0, 16, 16, 1, 1, 65, 0, 4, 0.1, 0)", "max_new = 65"),
    ("f('qe_attn_tree', 'pipllpllpppiiipifp', p, 0, 16, 8, 8, 16, 8, 8, 0, 16, 16, 1, 1, 1, 0, 3, 0.1, 0)", "3 heads over 2"),
    ("f('qe_attn_tree', 'pipllpllpppiiipifp', p, 0, 16, 8, 4, 16, 8, 8, 0, 16, 16, 1, 1, 1, 0, 4, 0.1, 0)", "strides of 8 elements"),
    ("f('qe_attn_prompt', 'pllpllpllpllppiiiiifip', *[16, 8, 8] * 4, 0, 16, 1, 1, 4, 2, 80, 0.1, 0, 0)", "qe_attn_prompt: d 80"),
    ("f('qe_attn_prompt', 'pllpllpllpllppiiiiifip', *[16, 8, 8] * 4, 0, 16, 1, 1, 4, 2, 64, -1.0, 0, 0)", "qe_attn_prompt: scale -1"),
    ("f('qe_attn_prompt', 'pllpllpllpllppiiiiifip', *[24, 8, 8] * 4, 0, 16, 1, 1, 4, 2, 64, 0.1, 0, 0)", "16-byte aligned"),
])
def test_entry_points_abort_with_check_message(code, msg):
    assert os.path.exists(LIB)
    r = subprocess.run([sys.executable, "-c", HEAD + code], capture_output=True, text=True, timeout=120)
    assert r.returncode != 0
    assert "check failed" in r.stderr and msg in r.stderr, r.stderr


@pytest.mark.parametrize("scale", [1e-46, 1e-39, 1e38, 1e39, float("inf")])
def test_scales_that_fp32_does_not_hold(scale):
    """too small or too large for the kernels' fp32 (the C-ABI would abort on what they become there)"""
    with pytest.raises(ValueError, match="scale"):
        ops.attn_prompt(z(4, 4, 64), z(4, 2, 64), z(4, 2, 64), i32(0, 4), scale=scale)
    with pytest.raises(ValueError, match="scale"):
        cache().attend(0, z(1, 4, 64), i32(0), i32(0, 1), 1, scale=scale)


def test_more_units_of_work_than_are_counted():
    c = cache(slots=1, max_tokens=1 << 30, page=1024)  # 2^25 units of 32 tokens, of 2 heads
    with pytest.raises(ValueError, match="not on|on a GPU"):
        c.attend(0, z(16, 4, 64), z(16, dtype=I32), z(17, dtype=I32), 64)
    with pytest.raises(ValueError, match="units of work"):
        c.attend(0, z(17, 4, 64), z(17, dtype=I32), z(18, dtype=I32), 64)
    with pytest.raises(ValueError, match="units of work"):
        c.attend(0, z(9, 6, 64), z(9, dtype=I32), z(10, dtype=I32), 64)  # 192 rows a head: two blocks
