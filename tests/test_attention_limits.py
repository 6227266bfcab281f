"""Sizes at the limits of the attention and cache entry points, refused by exceptions before the C-ABI would abort or cut them to
32 bits (CPU only)."""
import os
import subprocess
import sys

import pytest
import torch

from qengine_amd import ops
from test_abi import LIB
from test_attention_args import HEAD

BF, I32 = torch.bfloat16, torch.int32


def rows(n, heads, d=64):
    """n rows that take the memory of one"""
    return torch.zeros(1, heads, d, dtype=BF).expand(n, heads, d)


def i32(*v):
    return torch.tensor(v, dtype=I32)


def cache(layers=2):
    return ops.KVCache.empty(layers, 2, 16, 1, 64, 3, 32, device="cpu")


@pytest.mark.parametrize("n", [2 ** 30 + 1, 2 ** 31, 2 ** 32 + 4])
def test_more_rows_than_are_counted(n):
    with pytest.raises(ValueError, match="rows"):
        ops.attn_prompt(rows(n, 4), rows(n, 2), rows(n, 2), i32(0, 4))
    with pytest.raises(ValueError, match="rows"):
        cache().attend(0, rows(n, 1), i32(0), i32(0, 4), 4)
    with pytest.raises(ValueError, match="rows"):
        cache().append(0, rows(n, 1), rows(n, 1), i32(0), i32(0, 4))
    with pytest.raises(ValueError, match="rows"):
        cache().append(None, rows(n, 1)[None].expand(2, n, 1, 64), rows(n, 1)[None].expand(2, n, 1, 64), i32(0), i32(0, 4))


def test_the_most_rows_reach_the_gpu_check():
    n = 2 ** 30
    with pytest.raises(ValueError, match="on a GPU"):
        cache().append(0, rows(n, 1), rows(n, 1), i32(0), i32(0, 4))


ROWS = 2 ** 30 + 1


@pytest.mark.parametrize("code,msg", [
    (f"f('qe_kv_append', 'piipppppiip', p, 0, 1, 16, 16, 16, 16, 16, 1, {ROWS}, 0)", f"t {ROWS}"),
    (f"f('qe_attn_tree', 'pipllpllpppiiipifp', p, 0, 16, 8, 8, 16, 8, 8, 0, 16, 16, 1, {ROWS}, 1, 0, 4, 0.1, 0)", f"t = {ROWS}"),
    (f"f('qe_attn_prompt', 'pllpllpllpllppiiiiifip', *[16, 8, 8] * 4, 0, 16, 1, {ROWS}, 4, 2, 64, 0.1, 0, 0)", f"t {ROWS}"),
])
def test_entry_points_abort_with_check_message(code, msg):
    assert os.path.exists(LIB)
    r = subprocess.run([sys.executable, "-c", HEAD + code], capture_output=True, text=True, timeout=120)
    assert r.returncode != 0
    assert "check failed" in r.stderr and msg in r.stderr, r.stderr


def test_the_row_stride_of_one_row_is_not_passed_on(monkeypatch):
    """one row of a very wide buffer: its row stride is past what the C-ABI takes, and never used"""
    from qengine_amd import attention
    calls = []
    monkeypatch.setattr(attention, "_run", lambda at, name, sig, *a: calls.append((name, a)))
    wide = torch.empty_strided((1, 2, 64), (1 << 25, 64, 1), dtype=BF)
    q = torch.zeros(1, 4, 64, dtype=BF)
    ops.attn_prompt(q, wide, wide, i32(0, 1))
    (name, a), = calls
    assert name == "qe_attn_prompt" and a[4] < 1 << 24 and a[7] < 1 << 24


def test_more_layers_than_a_launch_takes():
    """append and accept would abort on them"""
    pool = torch.zeros(1, 2, 1, 16, 64, dtype=BF).expand(65536, 2, 1, 16, 64)
    ints = [torch.zeros(*x, dtype=I32) for x in ((3, 2), (3,), (3,), (2,))]
    ops.KVCache(pool[:65535], pool[:65535], *ints)
    with pytest.raises(ValueError, match="layers"):
        ops.KVCache(pool, pool, *ints)


@pytest.mark.parametrize("shape,strides", [((4, 4, 64), (0, 64, 1)), ((4, 4, 64), (256, 0, 1)), ((4, 4, 64), (64, 64, 1)), ((4, 4, 64), (128, 64, 1)),
                                           ((4, 4, 64), (256, 32, 1)), ((4, 4, 64), (64, 192, 1)), ((4, 1, 64), (32, 64, 1))])
def test_an_output_whose_rows_overlap(shape, strides):
    """expanded or overlapping outputs: which row's value stays would be a race"""
    out = torch.zeros(4096, dtype=BF).as_strided(shape, strides)
    heads = shape[1]
    with pytest.raises(ValueError, match="overlap"):
        ops.attn_prompt(rows(4, heads), rows(4, 1), rows(4, 1), i32(0, 4), out=out)
    with pytest.raises(ValueError, match="overlap"):
        cache().attend(0, rows(4, heads), i32(0), i32(0, 4), 4, out=out)


@pytest.mark.parametrize("shape,strides", [((4, 4, 64), (256, 64, 1)), ((4, 4, 64), (64, 256, 1)), ((4, 4, 64), (1024, 128, 1)), ((1, 4, 64), (0, 64, 1)),
                                           ((4, 1, 64), (64, 0, 1)), ((4, 4, 64), (64, 264, 1))])
def test_outputs_whose_rows_lie_apart(shape, strides):
    out = torch.zeros(4096, dtype=BF).as_strided(shape, strides)
    heads, n = shape[1], shape[0]
    with pytest.raises(ValueError, match="on a GPU"):
        ops.attn_prompt(rows(n, heads), rows(n, 1), rows(n, 1), i32(0, n), out=out)
    with pytest.raises(ValueError, match="on a GPU"):
        cache().attend(0, rows(n, heads), i32(0), i32(0, n), 4, out=out)
