"""What the entry points of 8-bit layers refuse, before anything reaches a GPU (CPU only): the wrappers by exceptions, the
C-ABI by the library's "check failed" message."""
import subprocess
import sys

import pytest
import torch

from qengine_amd import ops
from test_abi import LIB

BF, F16, F32, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64
F8 = torch.float8_e4m3fn


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def refused(call, a, change, error):
    a.update(change)
    with pytest.raises(error):
        call(**a)


@pytest.mark.parametrize("change,error", [
    (dict(x=z(4, 256, dtype=F32)), TypeError),
    (dict(x=z(256)), ValueError),
    (dict(x=z(256, 4).t()), ValueError),                      # columns apart
    (dict(x=z(4, 0), w=z(0, dtype=F32)), ValueError),
    (dict(x=z(4, 65537), w=z(65537, dtype=F32)), ValueError),
    (dict(w=z(256, dtype=F16)), TypeError),
    (dict(w=z(255, dtype=F32)), ValueError),
    (dict(w=z(512, dtype=F32)[::2]), ValueError),
    (dict(w=z(1, 256, dtype=F32)), ValueError),
    (dict(eps=0.0), ValueError),
    (dict(eps=-1e-6), ValueError),
    (dict(eps=float("nan")), ValueError),
    (dict(eps=float("inf")), ValueError),
    (dict(res=z(4, 256, dtype=F16)), TypeError),
    (dict(res=z(3, 256)), ValueError),
    (dict(res=z(256).expand(4, 256)), ValueError),            # written, and its rows are one
    (dict(res=z(4, 256), res_out=z(4, 255)), ValueError),
    (dict(res=z(4, 256), res_out=z(4, 256, dtype=F32)), TypeError),
    (dict(res_out=z(4, 256)), ValueError),
    (dict(out=z(4, 256, dtype=F32)), TypeError),
    (dict(out=z(4, 512)[:, ::2]), ValueError),
    (dict(out=z(4 * 256).as_strided((4, 256), (200, 1))), ValueError),
    (dict(), ValueError),                                     # all well, but not on a GPU
])
@pytest.mark.parametrize("f8", [False, True])
def test_norm_refusals(change, error, f8):
    refused(ops.rms_norm, dict(x=z(4, 256), w=z(256, dtype=F32), f8=f8), change, error)


@pytest.mark.parametrize("call,x,error", [
    (ops.quant_f8, z(4, 256, dtype=F32), TypeError),
    (ops.quant_f8, z(4), ValueError),
    (ops.quant_f8, z(4, 0), ValueError),
    (ops.quant_f8, z(8, 8).t(), ValueError),
    (ops.quant_f8, z(1).expand(4, (1 << 20) + 1), ValueError),
    (ops.quant_f8, z(1, 1).expand((1 << 23) + 1, 1), ValueError),
    (ops.silu_mul_f8, z(4, 255), ValueError),
    (ops.silu_mul_f8, z(4, 0), ValueError),
    (ops.silu_mul_f8, z(4, 256, dtype=torch.float64), TypeError),
    (ops.silu_mul_f8, z(4, 256), ValueError),                 # not on a GPU
])
def test_activation_refusals(call, x, error):
    with pytest.raises(error):
        call(x)


@pytest.mark.parametrize("q,s,error", [
    (z(32, 128), z(1, 1, dtype=F32), TypeError),
    (z(32, 128, dtype=F8), z(1, 1), TypeError),
    (z(32, 120, dtype=F8), z(1, 1, dtype=F32), ValueError),   # k not a multiple of 16
    (z(32, 256, dtype=F8), z(1, 1, dtype=F32), ValueError),
    (z(129, 128, dtype=F8), z(1, 1, dtype=F32), ValueError),
    (z(0, 128, dtype=F8), z(0, 1, dtype=F32), ValueError),
    (z(128, dtype=F8), z(1, dtype=F32), ValueError),
    (z(2, 32, 128, dtype=F8), z(1, 1, dtype=F32), ValueError),
    (z(1025, 1, 16, dtype=F8), z(1025, 1, 1, dtype=F32), ValueError),
    (z(32, 128, dtype=F8), z(1, 1, dtype=F32), ValueError),   # not on a GPU
])
def test_tile_refusals(q, s, error):
    with pytest.raises(error):
        ops.tile_f8(q, s)


def mat(experts=None, n=160, k=272):
    s = z(*((experts,) if experts else ()), 2, 3, dtype=F32)
    return ops.F8(z((experts or 1) * 10 * 3 * 2048, dtype=torch.uint8), s, n, k, experts or 1)


PRODUCT = [
    (dict(w=None), TypeError),
    (dict(q=z(4, 272)), TypeError),
    (dict(s=z(4, 3)), TypeError),
    (dict(q=z(4, 256, dtype=F8)), ValueError),
    (dict(q=z(272, dtype=F8)), ValueError),
    (dict(q=z(4, 280, dtype=F8)[:, :272]), ValueError),       # rows 280 apart
    (dict(q=z(4 * 272 + 1, dtype=F8)[1:].view(4, 272)), ValueError),
    (dict(s=z(4, 2, dtype=F32)), ValueError),
    (dict(s=z(3, 3, dtype=F32)), ValueError),
    (dict(s=z((3 << 22) + 3, dtype=F32).as_strided((4, 3), (1 << 22, 1))), ValueError),
    (dict(q=z(4 << 24, dtype=F8).as_strided((4, 272), (1 << 24, 1))), ValueError),
    (dict(dtype=F32), TypeError),
    (dict(y=z(4, 160, dtype=F32)), TypeError),
    (dict(y=z(4, 161)), ValueError),
    (dict(y=z(160, 4).t()), ValueError),
    (dict(y=z(160).expand(4, 160)), ValueError),
    (dict(), ValueError),
]


@pytest.mark.parametrize("change,error", PRODUCT + [(dict(w=mat(3)), ValueError)])
def test_product_refusals(change, error):
    refused(ops.matmul_f8, dict(w=mat(), q=z(4, 272, dtype=F8), s=z(4, 3, dtype=F32)), change, error)


@pytest.mark.parametrize("change,error", PRODUCT + [
    (dict(w=mat()), ValueError),
    (dict(off=z(4, dtype=I64)), TypeError),
    (dict(off=z(3, dtype=I32)), ValueError),
    (dict(off=z(8, dtype=I32)[::2]), ValueError),
    (dict(rows=z(4, dtype=I64)), TypeError),
    (dict(rows=z(2, 2, dtype=I32)), ValueError),
    (dict(rows=z(7, dtype=I32), y=z(4, 160)), ValueError),
])
def test_grouped_refusals(change, error):
    refused(ops.matmul_f8_grouped, dict(w=mat(3), q=z(4, 272, dtype=F8), s=z(4, 3, dtype=F32), off=z(4, dtype=I32)), change, error)


@pytest.mark.parametrize("change,error", [
    (dict(y=z(6, 64, dtype=torch.float64)), TypeError),
    (dict(y=z(64)), ValueError),
    (dict(y=z(6, 0)), ValueError),
    (dict(inv=z(6, dtype=I64)), TypeError),
    (dict(inv=z(5, dtype=I32)), ValueError),
    (dict(inv=z(3, 2, dtype=I32)), ValueError),
    (dict(w=z(3, 2)), TypeError),
    (dict(w=z(6, dtype=F32)), ValueError),
    (dict(w=z(2, 3, dtype=F32).t()), ValueError),
    (dict(w=z(1, 1025, dtype=F32), inv=z(1025, dtype=I32)), ValueError),
    (dict(add=z(3, 64, dtype=F16)), TypeError),
    (dict(add=z(2, 64)), ValueError),
    (dict(add=z(3, 64), out=z(3, 64, dtype=F32)), TypeError),
    (dict(out=z(3, 65)), ValueError),
    (dict(out=z(64).expand(3, 64)), ValueError),
    (dict(), ValueError),
])
def test_combine_refusals(change, error):
    refused(ops.moe_combine, dict(y=z(6, 64), inv=z(6, dtype=I32), w=z(3, 2, dtype=F32)), change, error)


BUF = z(64, 512)  # columns of one matrix are apart, shifted by less than a row they are not
LEFT, RIGHT, MID = BUF[:4, :256], BUF[:4, 256:], BUF[:4, 128:384]


@pytest.mark.parametrize("change,name", [
    (dict(x=LEFT, out=MID), "out overlaps x"),
    (dict(x=LEFT, out=BUF[1:5, :256]), "out overlaps x"),
    (dict(res=LEFT, out=LEFT), "out overlaps res"),
    (dict(res=z(4, 256), res_out=LEFT, out=LEFT), "out overlaps res_out"),
    (dict(res=MID, x=LEFT), "res_out overlaps x"),
    (dict(res=MID, res_out=LEFT), "res_out overlaps res"),
    (dict(x=LEFT, res=z(4, 256), res_out=LEFT, out=LEFT), "out overlaps res_out"),
    (dict(w=BUF[2, :256], out=LEFT), "out overlaps w"),
    (dict(w=BUF[2, 256:], out=LEFT), "out overlaps w"),  # between rows: refused too
    (dict(x=z(1, 256), res=BUF[2:3, :256], w=BUF[1:3].view(-1)[:512].view(F32)), "on a GPU"),
    (dict(x=z(1, 256), res=BUF[2:3, :256], w=BUF[1:3].view(-1)[2:514].view(F32)), "res_out overlaps w"),
    (dict(res=LEFT, res_out=BUF.view(128, 256)[:4]), "res_out overlaps res"),
    (dict(x=z(1, 256), res=BUF[2:3, :256], res_out=BUF.view(128, 256)[4:5]), "on a GPU"),
    (dict(x=LEFT, out=RIGHT), "on a GPU"),
    (dict(x=LEFT, out=LEFT), "on a GPU"),
    (dict(x=LEFT, out=BUF[4:8, :256]), "on a GPU"),
    (dict(x=LEFT, res=RIGHT), "on a GPU"),
    (dict(x=LEFT, res=RIGHT, res_out=LEFT), "on a GPU"),
    (dict(x=LEFT, res=LEFT), "on a GPU"),
    (dict(x=LEFT, res=RIGHT, out=LEFT), "on a GPU"),
])
def test_norm_overlaps(change, name):
    a = dict(x=z(4, 256), w=z(256))
    a.update(change)
    with pytest.raises(ValueError, match=name):
        ops.rms_norm(**a)


def test_product_and_combine_overlaps():
    q, s, off = z(4, 272, dtype=F8), z(4, 3, dtype=F32), z(4, dtype=I32)
    y = BUF[:4, :160]
    with pytest.raises(ValueError, match="y overlaps q"):
        ops.matmul_f8(mat(), BUF[:4, :136].view(F8), s, y=y)
    with pytest.raises(ValueError, match="y overlaps q"):
        ops.matmul_f8_grouped(mat(3), BUF[:4, 80:216].view(F8), s, off, y=y)
    with pytest.raises(ValueError, match="y overlaps s"):
        ops.matmul_f8(mat(), q, BUF[:4, 150:156].view(F32), y=y)
    with pytest.raises(ValueError, match="y overlaps off"):
        ops.matmul_f8_grouped(mat(3), q, s, BUF[0, :8].view(I32), y=y)
    with pytest.raises(ValueError, match="on a GPU"):
        ops.matmul_f8(mat(), BUF[:4, 160:296].view(F8), s, y=y)
    inv, w = z(6, dtype=I32), z(3, 2, dtype=F32)
    for add, out, name in [(None, BUF[:3, :64], "overlaps y"), (BUF[8:11, :64], BUF[9:12, :64], "overlaps add"),
                           (BUF[8:11, :64], BUF[8:11, :64], "on a GPU"), (None, BUF[:3, 64:128], "on a GPU")]:
        with pytest.raises(ValueError, match=name):
            ops.moe_combine(BUF[:6, :64], inv, w, add=add, out=out)


@pytest.mark.parametrize("change,error", [
    (dict(q=z(10 * 3 * 2048 - 16, dtype=torch.uint8)), ValueError),
    (dict(q=z(10 * 3 * 2048, dtype=F8)), TypeError),
    (dict(q=z(10 * 3 * 2048 + 1, dtype=torch.uint8)[1:]), ValueError),
    (dict(q=z(10 * 3 * 4096, dtype=torch.uint8)[::2]), ValueError),
    (dict(s=z(2, 3)), TypeError),
    (dict(s=z(3, 2, dtype=F32)), ValueError),
    (dict(s=z(3, 2, dtype=F32).t()), ValueError),
    (dict(s=z(2, 2, 3, dtype=F32)), ValueError),
    (dict(n=177), ValueError),
    (dict(k=400), ValueError),
    (dict(experts=2), ValueError),
])
def test_weights_by_hand(change, error):
    a = dict(q=z(10 * 3 * 2048, dtype=torch.uint8), s=z(2, 3, dtype=F32), n=160, k=272)
    ops.F8(**a)
    refused(ops.F8, a, change, error)


@pytest.mark.parametrize("n,k,experts", [(160, 264, 1), (0, 272, 1), (160, 0, 1), (-5, 272, 1), ((1 << 20) + 1, 16, 1), (16, (1 << 20) + 16, 1),
                                         (16, 16, 1025), (16, 16, 0), (16, 16, -1)])
def test_weights_by_hand_of_sizes_that_no_product_takes(n, k, experts):
    """the sizes that the library would end the process for"""
    bn, bk = max(-(-n // 128), 0), max(-(-k // 128), 0)
    q, s = z(max(experts, 0) * max(-(-n // 16), 0) * bk * 2048, dtype=torch.uint8), z(max(experts, 0), bn, bk, dtype=F32)
    with pytest.raises(ValueError, match="at most"):
        ops.F8(q, s, n, k, experts)


@pytest.mark.parametrize("bt,bw,parts", [(16, 0, 4), (48, 64, 1), (64, 256, 1), (256, 128, 1), (64, 128, 0), (256, 256, 17)])
def test_choices(bt, bw, parts):
    with pytest.raises(ValueError, match="no blocks"):
        ops.matmul_f8_choice(mat(), z(4, 272, dtype=F8), z(4, 3, dtype=F32), bt, bw, parts)


@pytest.mark.parametrize("bw", [0, 32, 1 << 20])
def test_choices_of_few_rows_whatever_the_columns(bw):
    """blocks of 16 rows have 32 columns: too many of them end the process in the library"""
    t, n = 1 << 17, 1 << 17
    w = ops.F8(z(n // 16 * 2048, dtype=torch.uint8), z(n // 128, 1, dtype=F32), n, 16)
    with pytest.raises(ValueError, match="rows of 131072 in"):
        ops.matmul_f8_choice(w, z(t, 16, dtype=F8), z(t, 1, dtype=F32), 16, bw, 1)


@pytest.mark.parametrize("change,error,match", [
    (dict(bt=32), ValueError, "no blocks of 32"),
    (dict(bt=0), ValueError, "no blocks of 0"),
    (dict(q=z(0, 272, dtype=F8), s=z(0, 3, dtype=F32)), ValueError, "for 0 of 0 rows"),
    (dict(w=mat()), ValueError, "of them for matmul_f8_grouped"),
    (dict(off=z(4, dtype=I64)), TypeError, "off"),
    (dict(rows=z(2, 2, dtype=I32)), ValueError, "rows"),
    (dict(y=z(4, 161)), ValueError, "y has shape"),
    (dict(q=z(1, 272, dtype=F8).expand(1 << 24, 272), s=z(1, 3, dtype=F32).expand(1 << 24, 3), rows=z(4, dtype=I32)), ValueError, "on a GPU"),
    (dict(), ValueError, "on a GPU"),
])
def test_grouped_choice_refusals(change, error, match):
    a = dict(w=mat(3), q=z(4, 272, dtype=F8), s=z(4, 3, dtype=F32), off=z(4, dtype=I32), bt=256)
    a.update(change)
    with pytest.raises(error, match=match):
        ops.matmul_f8_grouped_choice(**a)


@pytest.mark.parametrize("call,msg", [
    ("qe_rms_norm(P, L(8), None, L(0), None, L(0), P, F(1e-6), P, L(8), None, L(0), None, L(0), L(0), 0, 8, 0, None)", "rms_norm: 0 rows of 8"),
    ("qe_rms_norm(P, L(8), None, L(0), None, L(0), P, F(1e-6), P, L(8), None, L(0), None, L(0), L(0), 1, 65537, 0, None)", "1 rows of 65537"),
    ("qe_rms_norm(P, L(8), P, L(8), None, L(0), P, F(1e-6), P, L(8), None, L(0), None, L(0), L(0), 1, 8, 0, None)", "a tensor is missing"),
    ("qe_rms_norm(P, L(8), None, L(0), None, L(0), P, F(1e-6), None, L(8), None, L(0), None, L(0), L(0), 1, 8, 0, None)", "a tensor is missing"),
    ("qe_rms_norm(P, L(8), None, L(0), None, L(0), P, F(0), P, L(8), None, L(0), None, L(0), L(0), 1, 8, 0, None)", "eps 0"),
    ("qe_rms_norm(P, L(8), None, L(0), None, L(0), P, F(1e-6), P, L(8), None, L(0), None, L(0), L(0), 1, 8, 2, None)", "flags 2"),
    ("qe_act_f8(P, L(8), 0, P, L(8), P, L(1), L(1), -1, 8, 0, None)", "act_f8: -1 rows"),
    ("qe_act_f8(P, L(8), 0, P, L(8), P, L(1), L(1), 1 << 24, 4096, 0, None)", "too many for a call"),
    ("qe_act_f8(P, L(8), 0, P, L(8), None, L(1), L(1), 1, 8, 0, None)", "a tensor is missing"),
    ("qe_tile_f8(P, L(8), L(0), 16, 24, 1, P, None)", "tile_f8: n = 16, k = 24"),
    ("qe_tile_f8(P, L(24), L(0), 16, 32, 1, P, None)", "alignment"),
    ("qe_tile_f8(P, L(32), L(0), 16, 32, 1025, P, None)", "1025 matrices"),
    ("qe_matmul_f8(P, P, 16, 24, P, L(32), P, L(1), L(1), 1, P, L(16), 0, None)", "matmul_f8: n = 16, k = 24"),
    ("qe_matmul_f8(P, P, 16, 32, P, L(40), P, L(1), L(1), 1, P, L(16), 0, None)", "16-byte aligned"),
    ("qe_matmul_f8(P, P, 16, 32, P, L(32), P, L(1), L(1), 0, P, L(16), 0, None)", "0 rows of x"),
    ("qe_matmul_f8(P, P, 16, 32, P, L(32), P, L(1), L(1), 1, P, L(16), 2, None)", "flags 2"),
    ("qe_matmul_f8(P, P, 1 << 20, 32, P, L(32), P, L(1), L(1), 1 << 24, P, L(1 << 20), 0, None)", "too many for a call"),
    ("qe_matmul_f8_grouped(P, P, 16, 32, 2, P, L(32), P, L(1), L(1), 4, None, None, 4, P, L(16), 0, None)", "off is missing"),
    ("qe_matmul_f8_grouped(P, P, 16, 32, 2, P, L(32), P, L(1), L(1), 4, P, None, 5, P, L(16), 0, None)", "5 rows of y, 4 of x"),
    ("qe_matmul_f8_grouped(P, P, 16, 32, 0, P, L(32), P, L(1), L(1), 4, P, None, 4, P, L(16), 0, None)", "0 matrices"),
    ("qe_matmul_f8_grouped_choice(P, P, 16, 32, 2, P, L(32), P, L(1), L(1), 4, P, None, 4, P, L(16), 0, 32, None)", "blocks of 32 rows"),
    ("qe_matmul_f8_grouped_choice(P, P, 16, 32, 2, P, L(32), P, L(1), L(1), 4, None, None, 4, P, L(16), 0, 64, None)", "off is missing"),
    ("qe_matmul_f8_grouped_choice(P, P, 16, 32, 2, P, L(1 << 20), P, L(1), L(1), 4096, P, P, 4, P, L(16), 0, 256, None)", "blocks of 256 rows"),
    ("qe_matmul_f8_grouped_choice(P, P, 16, 32, 2, P, L(32), P, L(1), L(1), 4, P, None, 5, P, L(16), 0, 64, None)", "5 rows of y, 4 of x"),
    ("qe_moe_combine(P, L(8), 4, P, P, None, L(0), P, L(8), 2, 2000, 8, 0, 0, None)", "2000 rows each"),
    ("qe_moe_combine(P, L(8), 4, P, P, None, L(0), P, L(8), 2, 2, 8, 0, 2, None)", "y's type or fp32"),
    ("qe_moe_combine(P, L(8), 4, P, P, None, L(0), P, L(8), 2, 2, 8, 18, 2, None)", "flags 18"),
    ("qe_moe_combine(P, L(8), 4, None, P, None, L(0), P, L(8), 2, 2, 8, 0, 0, None)", "a tensor is missing"),
])
def test_c_refusals(call, msg):
    code = (f"import ctypes; lib = ctypes.CDLL({LIB!r}); P, L, F = ctypes.c_void_p(4096), ctypes.c_int64, ctypes.c_float; lib.{call}")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert r.returncode != 0 and "check failed" in r.stderr and msg in r.stderr, r.stderr
