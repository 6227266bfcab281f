"""The norm, the activation and the combine of 8-bit layers against their formulas in 64 bits (bounds: f8_ref.py)."""
import pytest
import torch

import f8_ref as ref
from qengine_amd import ops

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rows(dev, t, d, dtype, seed, size=1.0, pad=0):
    g = ref.gen(dev, seed)
    x = torch.randn(t, d + pad, device=dev, generator=g) * torch.exp(torch.randn(d + pad, device=dev, generator=g)) * size
    return x.to(dtype)[:, :d]


# every number of threads and chunks a row, odd ends, a group that ends inside a chunk
DIMS = [1, 7, 8, 127, 128, 129, 136, 512, 520, 1000, 2048, 2049, 2880, 4096, 5120, 8200, 16384, 16392, 33000, 65536]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", DIMS)
def test_norm(dev, d, dtype):
    x, r = rows(dev, 3, d, dtype, d), rows(dev, 3, d, dtype, d + 1)
    g = ref.gen(dev, d + 2)
    w = 1 + 0.3 * torch.randn(d, device=dev, generator=g)
    y = ops.rms_norm(x, w, 1e-6)
    ref.check_16(y, ref.norm(x, w, 1e-6), ref.NORM, "16 bits")
    q, s = ops.rms_norm(x, w, 1e-6, f8=True)
    ref.check_quantized(q, s, ref.norm(x, w, 1e-6), ref.NORM, "8 bits")
    h = torch.empty_like(x)
    y2 = torch.empty_like(x)
    kept = r.clone()
    q, s = ops.rms_norm(x, w.to(dtype), 1e-5, res=r, res_out=h, out=y2, f8=True)
    want = (x.float() + r.float()).to(dtype)
    assert torch.equal(h, want) and torch.equal(r, kept)
    ref.check_16(y2, ref.norm(want, w.to(dtype), 1e-5), ref.NORM, "both, 16 bits")
    ref.check_quantized(q, s, ref.norm(want, w.to(dtype), 1e-5), ref.NORM, "both, 8 bits")
    assert ops.rms_norm(x, w.to(dtype), 1e-5, res=r, out=x) is x  # in place: the stream and the row
    assert torch.equal(r, want) and torch.equal(x, y2)


@pytest.mark.parametrize("t", [1, 2, 63, 500])
@pytest.mark.parametrize("d,pad", [(256, 8), (256, 3), (1536, 16), (770, 1)])
def test_norm_strides(dev, t, d, pad):
    x, r = rows(dev, t, d, BF, 1, pad=pad), rows(dev, t, d, BF, 2, pad=2 * pad)
    w = torch.ones(d, device=dev)
    room = torch.full((t, d + 5 * pad), 7.0, dtype=BF, device=dev)
    out = room[:, :d]
    q, s = ops.rms_norm(x, w, res=r, out=out, f8=True)
    h = r.clone()
    ref.check_16(out, ref.norm(h, w, 1e-6), ref.NORM)
    ref.check_quantized(q, s, ref.norm(h, w, 1e-6), ref.NORM)
    assert (room[:, d:] == 7).all()


@pytest.mark.parametrize("dtype", [BF, F16])
def test_norm_far_values(dev, dtype):
    """rows of the type's largest values, of its least, of zeros: finite; infinities and NaN stay in their rows"""
    big = torch.finfo(dtype).max
    x = rows(dev, 8, 640, dtype, 3)
    x[0], x[1], x[2] = big, -big, 0
    x[3, 5], x[4] = big, torch.finfo(dtype).tiny
    x[5, 7], x[6, 9] = float("inf"), float("nan")
    w = torch.ones(640, device=dev)
    y = ops.rms_norm(x, w, 1e-6)
    fine = [0, 1, 2, 3, 4, 7]
    ref.check_16(y[fine], ref.norm(x[fine], w, 1e-6), ref.NORM)
    assert y[5, 7].isnan() and (y[5, 8:] == 0).all() and y[6].isnan().all()
    q, s = ops.rms_norm(x, w, 1e-6, f8=True)
    ref.check_quantized(q[fine], s[fine], ref.norm(x[fine], w, 1e-6), ref.NORM)
    assert (q[2].float() == 0).all() and (s[2] > 0).all() and q[6].float().isnan().all()


def test_norm_far_values_and_eps(dev):
    x = torch.zeros(2, 65536, device=dev, dtype=BF)
    x[:, 5] = 2.0 ** 64  # the mean of the squares: 2^112
    w = torch.ones(65536, device=dev)
    q, s = ops.rms_norm(x, w, 2.0 ** 100, f8=True)
    ref.check_quantized(q, s, ref.norm(x, w, 2.0 ** 100), ref.NORM)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("t,d", [(1, 1), (1, 5120), (3, 127), (5, 128), (17, 129), (33, 640), (9, 1000), (2, 2048), (3, 2056), (2, 17408), (300, 72), (1, 65537)])
def test_quantized(dev, t, d, dtype):
    x = rows(dev, t, d, dtype, d)
    q, s = ops.quant_f8(x)
    ref.check_quantized(q, s, x.double(), 0, "rows")
    x = rows(dev, t, 2 * d, dtype, d + 1, 2.0)
    q, s = ops.silu_mul_f8(x)
    ref.check_quantized(q, s, ref.silu_mul(x), ref.SILU, "silu")


def test_quantized_strides(dev):
    for pad in (1, 8):
        x = rows(dev, 40, 400, BF, 5, pad=pad)
        ref.check_quantized(*ops.quant_f8(x), x.double(), 0)
        ref.check_quantized(*ops.silu_mul_f8(x), ref.silu_mul(x), ref.SILU)
        odd = rows(dev, 40, 401, BF, 6, pad=pad)[:, 1:]  # not aligned
        ref.check_quantized(*ops.quant_f8(odd), odd.double(), 0)


def test_quantized_exactly(dev):
    """where the scale is a power of two, the bytes are torch's"""
    g = ref.gen(dev, 4)
    x = (torch.randn(64, 256, device=dev, generator=g) * 60).clamp(-440, 440).to(BF)
    x[:, 0], x[:, 200] = 448, -448
    q, s = ops.quant_f8(x)
    assert torch.equal(q.view(torch.uint8), x.to(ref.F8).view(torch.uint8)) and (s == 1).all()


def test_quantized_far_values(dev):
    x = rows(dev, 6, 512, BF, 7)
    x[0], x[1] = 0, torch.finfo(BF).max
    x[2] = 2.0 ** -133
    x[3, 130], x[4, 260] = float("inf"), float("nan")
    q, s = ops.quant_f8(x)
    ref.check_quantized(q[:3], s[:3], x[:3].double(), 0)
    assert (q[0].float() == 0).all() and s.isnan().sum() == 0
    assert s[3, 1].isinf() and q[3, 130].float().isnan() and q[3].float().isnan().sum() == 1
    assert q[4, 260].float().isnan() and q[4].float().isnan().sum() == 1
    ref.check_quantized(q[3, :128][None], s[3, :1][None], x[3, :128][None].double(), 0)
    x = torch.zeros(4, 256, device=dev, dtype=BF)
    x[:, 128:] = 1
    x[0, :128], x[1, :128], x[2, :128], x[3, :128] = -1e4, 1e4, -3e38, -88.5  # silu: 0, the value, 0, next to 0
    q, s = ops.silu_mul_f8(x)
    ref.check_quantized(q, s, ref.silu_mul(x), ref.SILU)


@pytest.mark.parametrize("gate", [3.3e38, 2.4e38, 1e38, 200.0, 88.0, 87.0, -87.0, -88.0, -200.0, -1e38, -3.3e38])
def test_silu_of_far_values(dev, gate):
    x = torch.full((2, 256), gate, device=dev, dtype=BF)
    x[:, 128:] = torch.linspace(-0.9, 0.9, 128, device=dev)
    q, s = ops.silu_mul_f8(x)
    ref.check_quantized(q, s, ref.silu_mul(x), ref.SILU)


def test_silu_of_infinity(dev):
    x = torch.ones(1, 512, device=dev, dtype=BF)
    x[0, 3] = float("inf")
    q, s = ops.silu_mul_f8(x)
    assert s[0, 0].isinf() and q[0, 3].float().isnan() and q[0].float().isnan().sum() == 1
    ref.check_quantized(q[:, 128:], s[:, 1:], ref.silu_mul(torch.ones(1, 256, device=dev)), ref.SILU)


@pytest.mark.parametrize("dtype,otype", [(BF, BF), (F16, F16), (F32, F32), (BF, F32), (F16, F32)])
@pytest.mark.parametrize("t,topk,d", [(1, 1, 1), (1, 10, 2048), (7, 3, 129), (64, 8, 640), (5, 1, 4100), (3, 0, 16), (300, 2, 72)])
def test_combine(dev, t, topk, d, dtype, otype):
    g = ref.gen(dev, t + d)
    slots = max(1, t * topk)
    y = rows(dev, slots, d, dtype, 1)
    inv = torch.randperm(slots, device=dev, generator=g).int()[:t * topk]
    w = torch.rand(t, topk, device=dev, generator=g) - 0.2
    add = rows(dev, t, d, otype, 2)
    terms = w[..., None].double() * y[inv.long()].double().view(t, topk, d)
    for more in (None, add):
        if more is None and otype != dtype:
            out = torch.empty(t, d, dtype=otype, device=dev)
            assert ops.moe_combine(y, inv, w, out=out) is out
        else:
            out = ops.moe_combine(y, inv, w, add=more)
        assert out.dtype == (otype if more is not None or otype != dtype else dtype)
        want, size = terms.sum(1), terms.abs().sum(1)
        if more is not None:
            want, size = want + more.double(), size + more.double().abs()
        off = (topk + 1) * ref.U * size
        ref.within(out, want, off + ref.half(out.dtype, want.abs() + off))
    assert ops.moe_combine(y, inv, w, add=add, out=add) is add and torch.equal(add, out)


def test_combine_skips_bad_rows(dev):
    y = torch.ones(4, 64, device=dev)
    inv = torch.tensor([0, 4, -1, 3, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)
    w = torch.tensor([[1.0, 2.0], [4.0, 8.0], [16.0, 32.0]], device=dev)
    assert ops.moe_combine(y, inv, w).tolist() == [[1.0] * 64, [8.0] * 64, [0.0] * 64]


def test_no_rows(dev):
    x = torch.empty(0, 256, dtype=BF, device=dev)
    assert ops.rms_norm(x, torch.ones(256, device=dev)).shape == (0, 256)
    q, s = ops.quant_f8(x)
    assert q.shape == (0, 256) and s.shape == (0, 2)
    assert ops.moe_combine(torch.ones(1, 8, device=dev), torch.empty(0, dtype=torch.int32, device=dev), torch.empty(0, 2, device=dev)).shape == (0, 8)


def test_large(dev):
    """values beyond 2^32 bytes: the last rows"""
    t, d = 40000, 65536
    x = torch.zeros(t, d, dtype=BF, device=dev)
    x[-3:] = rows(dev, 3, d, BF, 1)
    w = torch.ones(d, device=dev)
    y = ops.rms_norm(x, w)
    ref.check_16(y[-3:], ref.norm(x[-3:], w, 1e-6), ref.NORM)
    assert (y[-4] == 0).all()
    del y
    q, s = ops.rms_norm(x, w, f8=True)
    ref.check_quantized(q[-3:], s[-3:], ref.norm(x[-3:], w, 1e-6), ref.NORM)
    q, s = ops.silu_mul_f8(x)
    ref.check_quantized(q[-3:], s[-3:], ref.silu_mul(x[-3:]), ref.SILU)
    inv = torch.tensor([t - 1, t - 2, t - 3, 5], dtype=torch.int32, device=dev)
    weight = torch.tensor([[0.5, 2.0], [1.0, 1.0]], device=dev)
    out = ops.moe_combine(x, inv, weight)
    v = x[-3:].double()
    want = torch.stack([0.5 * v[2] + 2 * v[1], v[0]])
    size = torch.stack([0.5 * v[2].abs() + 2 * v[1].abs(), v[0].abs()])
    ref.within(out, want, 3 * ref.U * size + ref.half(BF, want.abs() + 3 * ref.U * size))


@pytest.mark.parametrize("gate", [-43.0, -44.25, -45.0, -60.0, -80.0, -87.0, -87.5, -88.0, -88.5, -89.0, -95.0, -120.0, -150.0, -170.0])
def test_silu_of_far_gates_and_large_values(dev, gate):
    """exp(-gate) at the end of fp32 and beyond, silu(gate) * up not: alone, and among usual values"""
    g = ref.gen(dev, int(-4 * gate))
    x = rows(dev, 4, 1024, BF, 3)
    up = torch.exp2(torch.rand(4, 512, device=dev, generator=g) * 27 + 100) * torch.where(torch.rand(4, 512, device=dev, generator=g) < 0.5, -1, 1)
    x[:2, :512], x[:2, 512:] = gate, up[:2]
    few = torch.rand(4, 512, device=dev, generator=g) < 0.1
    few[:2] = False
    x[:, :512][few], x[:, 512:][few] = gate, up.to(BF)[few]
    q, s = ops.silu_mul_f8(x)
    ref.check_quantized(q, s, ref.silu_mul(x), ref.SILU)


@pytest.mark.parametrize("size", [2.0 ** -66, 2.0 ** -50, 2.0 ** -20, 1.0])
def test_norm_of_small_values_in_a_far_row(dev, size):
    """a row whose squares leave fp32 keeps what its small values are"""
    g = ref.gen(dev, 5)
    x = (size * (1 + torch.rand(3, 640, device=dev, generator=g))).to(BF)
    x[:, 5] = 2.0 ** 64
    for scale in (1.0, 2.0 ** 60):
        w = torch.full((640,), scale, device=dev)
        y = torch.empty_like(x)
        q, s = ops.rms_norm(x, w, 1e-6, out=y, f8=True)
        ref.check_16(y, ref.norm(x, w, 1e-6), ref.NORM)
        ref.check_quantized(q, s, ref.norm(x, w, 1e-6), ref.NORM)


def padded(dev, t, d, dtype, seed, pad):
    """rows with `pad` columns of sevens behind each -> the rows, and what holds them"""
    room = torch.full((t, d + pad), 7.0, dtype=dtype, device=dev)
    room[:, :d] = rows(dev, t, d, dtype, seed)
    return room[:, :d], room


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("t", [1, 2, 63, 500])
@pytest.mark.parametrize("d,pads", [(256, (8, 16, 24, 40)), (256, (3, 5, 1, 7)), (1536, (16, 0, 8, 64)), (770, (1, 2, 3, 4))])
def test_norm_rows_apart(dev, t, d, pads, dtype):
    """x, the stream, its next buffer and the output each with rows of their own distance"""
    (x, xr), (r, rr), (h, hr), (y, yr) = (padded(dev, t, d, dtype, i, p) for i, p in enumerate(pads))
    kept, room = r.clone(), rr.clone()
    w = 1 + 0.3 * torch.randn(d, device=dev, generator=ref.gen(dev, 9))
    want = (x.float() + kept.float()).to(dtype)
    q, s = ops.rms_norm(x, w, res=r, res_out=h, out=y, f8=True)
    assert torch.equal(h, want) and torch.equal(rr, room)
    ref.check_16(y, ref.norm(want, w, 1e-6), ref.NORM)
    ref.check_quantized(q, s, ref.norm(want, w, 1e-6), ref.NORM)
    for v in (xr, rr, hr, yr):
        assert (v[:, d:] == 7).all()
    ops.rms_norm(x, w, res=r, out=y)  # the stream in place
    assert torch.equal(r, want) and (rr[:, d:] == 7).all() and (yr[:, d:] == 7).all()
    ref.check_16(y, ref.norm(want, w, 1e-6), ref.NORM)
    r.copy_(kept)
    x2 = x.clone()
    q2, s2 = ops.rms_norm(x, w, res=r, res_out=x, f8=True)  # into x
    assert torch.equal(x, want) and torch.equal(r, kept) and (xr[:, d:] == 7).all()
    assert torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)
    x.copy_(x2)
    ref.check_16(ops.rms_norm(x, w), ref.norm(x, w, 1e-6), ref.NORM)


@pytest.mark.parametrize("dtype,otype", [(BF, BF), (F16, F32), (F32, F32)])
@pytest.mark.parametrize("t,topk,d", [(1, 10, 256), (7, 3, 129), (64, 8, 640), (300, 2, 72)])
@pytest.mark.parametrize("pads", [(8, 16, 24), (3, 5, 1), (0, 8, 5)])
def test_combine_rows_apart(dev, t, topk, d, pads, dtype, otype):
    """the experts' rows, what they are added to and the output each with rows of their own distance"""
    g = ref.gen(dev, t + d)
    (y, yr), (add, ar), (out, outr) = padded(dev, t * topk, d, dtype, 1, pads[0]), padded(dev, t, d, otype, 2, pads[1]), padded(dev, t, d, otype, 3, pads[2])
    inv = torch.randperm(t * topk, device=dev, generator=g).int()
    w = torch.rand(t, topk, device=dev, generator=g) - 0.2
    terms = w[..., None].double() * y[inv.long()].double().view(t, topk, d)
    for more in (add, None):
        kept = ar.clone()
        assert ops.moe_combine(y, inv, w, add=more, out=out) is out
        assert torch.equal(ar, kept) and (outr[:, d:] == 7).all() and (yr[:, d:] == 7).all()
        want, size = terms.sum(1), terms.abs().sum(1)
        if more is not None:
            want, size = want + more.double(), size + more.double().abs()
        off = (topk + 1) * ref.U * size
        ref.within(out, want, off + ref.half(otype, want.abs() + off))


@pytest.mark.parametrize("pads", [(8, 16), (3, 5)])
def test_activation_rows_apart(dev, pads):
    for pad in pads:
        x, room = padded(dev, 90, 816, BF, 4, pad)
        ref.check_quantized(*ops.silu_mul_f8(x), ref.silu_mul(x.contiguous()), ref.SILU)
        ref.check_quantized(*ops.quant_f8(x), x.double(), 0)
        assert (room[:, 816:] == 7).all()
