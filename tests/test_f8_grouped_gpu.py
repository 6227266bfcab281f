"""Products grouped by expert, by each of their kernels whatever the sizes would choose (bounds: f8_ref.py)."""
import pytest
import torch

import f8_ref as ref
from qengine_amd import ops

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16
KERNELS = [16, 64, 128, 256]  # rows a block
# around every bound of a block of 256 rows, empty segments at the ends and inside, one row
LENS = [[1], [0, 256, 0], [255, 257, 1], [700, 0, 513, 256, 0, 0], [3, 5, 0, 2, 600], [0] * 30 + [5] + [0] * 33 + [300], [0, 0]]


def rows_of(x, at):
    return x.view(torch.uint8)[at].view(ref.F8)


def starts(dev, lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


@pytest.mark.parametrize("gather", [None, 9, 400])
@pytest.mark.parametrize("n,k", [(640, 512), (65, 208), (258, 2064)])
@pytest.mark.parametrize("lens", LENS, ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("bt", KERNELS)
def test_segments(dev, bt, lens, n, k, gather):
    """ragged and empty segments between rows that belong to none, in order and by index, both types"""
    first, tail, e = 2, 3, len(lens)
    r = first + sum(lens) + tail
    t = gather or r
    q, s = ref.weights(dev, (e, n, k), 1)
    x, xs = ref.activations(dev, t, k, 2, pad=16)
    off, w = starts(dev, lens, first), ops.tile_f8(q, s)
    rows = torch.randint(t, (r,), device=dev, generator=ref.gen(dev, 3)).int() if gather else None
    for dtype, more in ((BF, 0), (F16, 5)):
        room = torch.full((r, n + more), 7.0, dtype=dtype, device=dev)
        y = room[:, :n]
        assert ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=rows, y=y) is y
        assert (y[:first] == 7).all() and (y[r - tail:] == 7).all() and (room[:, n:] == 7).all()
        c = off.tolist()
        for i in range(e):
            if lens[i]:
                at = torch.arange(c[i], c[i + 1], device=dev) if rows is None else rows[c[i]:c[i + 1]].long()
                ref.check_product(y[c[i]:c[i + 1]], rows_of(x, at), xs[at], q[i], s[i], f"segment {i} of {lens[i]}")


@pytest.mark.parametrize("n,k", [(640, 1024), (257, 400)])
@pytest.mark.parametrize("bt", KERNELS)
def test_whole_numbers(dev, bt, n, k):
    """every product and sum is exact, so the output is the sum rounded once; scales of every row and block differ"""
    lens = [300, 0, 17, 256, 90]
    g, r, e = ref.gen(dev, n), sum(lens), len(lens)
    x = torch.randint(-8, 9, (50, k), device=dev, generator=g).float().to(ref.F8)
    q = torch.randint(-8, 9, (e, n, k), device=dev, generator=g).float().to(ref.F8)
    xs = torch.exp2(torch.randint(-3, 1, (50, -(-k // 128)), device=dev, generator=g).float())
    s = torch.exp2(torch.randint(-3, 1, (e, -(-n // 128), -(-k // 128)), device=dev, generator=g).float())
    rows = torch.randint(50, (r,), device=dev, generator=g).int()
    off, at, w = starts(dev, lens), rows.long(), ops.tile_f8(q, s)
    c = off.tolist()
    want = torch.cat([ref.product(rows_of(x, at[c[i]:c[i + 1]]), xs[at[c[i]:c[i + 1]]], q[i], s[i])[0] for i in range(e) if lens[i]])
    for dtype in (BF, F16):
        assert torch.equal(ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=rows, dtype=dtype), want.to(dtype))
        assert torch.equal(ops.matmul_f8_grouped_choice(w, rows_of(x, at), xs[at], off, bt, dtype=dtype), want.to(dtype))


@pytest.mark.parametrize("lens,n,k", [([5, 0, 9], 97, 272), ([300, 0, 260], 640, 512), ([2100, 900], 1024, 400)])
@pytest.mark.parametrize("bt", KERNELS)
def test_bad_indexes(dev, bt, lens, n, k):
    """an index outside x: as row 0, but zeros, whatever row 0 holds"""
    r, t = sum(lens), 50
    q, s = ref.weights(dev, (len(lens), n, k), 1)
    x, xs = ref.activations(dev, t, k, 2)
    off, w, g = starts(dev, lens), ops.tile_f8(q, s), ref.gen(dev, r)
    rows = torch.randint(1, t, (r,), device=dev, generator=g).int()
    bad = torch.rand(r, device=dev, generator=g) < 0.3
    bad[0] = bad[-1] = True
    far = torch.tensor([-1, t, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)[torch.arange(r, device=dev) % 4]
    want = ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=torch.where(bad, 0, rows))
    y = ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=torch.where(bad, far, rows))
    assert torch.equal(y, torch.where(bad[:, None], 0, want))
    x, xs = x.clone(), xs.clone()
    x.view(torch.uint8)[0], xs[0] = 0x7F, float("inf")
    assert torch.equal(ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=torch.where(bad, far, rows)), y)
    assert (ops.matmul_f8_grouped_choice(w, x[:0], xs[:0], off, bt, rows=rows) == 0).all()


@pytest.mark.parametrize("bt", KERNELS)
def test_bad_segments(dev, bt):
    """segments that do not ascend or leave y write nothing outside"""
    q, s = ref.weights(dev, (4, 96, 128), 1)
    x, xs = ref.activations(dev, 6, 128, 2)
    w = ops.tile_f8(q, s)
    for bad in ([3, 1, 9, 2, 4], [-5, 2, 2, 100, 3], [2 ** 31 - 1, 0, 0, 0, -2 ** 31], [0, 6, 0, 6, 0]):
        room = torch.full((20, 96), 7.0, dtype=BF, device=dev)
        ops.matmul_f8_grouped_choice(w, x, xs, torch.tensor(bad, dtype=torch.int32, device=dev), bt, y=room[7:13])
        assert (room[:7] == 7).all() and (room[13:] == 7).all()


@pytest.mark.parametrize("bt", KERNELS)
def test_values_stay_in_their_rows(dev, bt):
    """a NaN or an infinite scale spoils its row or its columns, in its own segment"""
    lens, n, k = [40, 300, 7], 300, 528
    q, s = ref.weights(dev, (3, n, k), 5)
    x, xs = ref.activations(dev, sum(lens), k, 6)
    x, xs = x.contiguous(), xs.clone()
    x.view(torch.uint8)[45, 520] = 0x7F
    xs[50, 4] = float("inf")
    q.view(torch.uint8)[1, 7, 3] = 0xFF
    y = ops.matmul_f8_grouped_choice(ops.tile_f8(q, s), x, xs, starts(dev, lens), bt, dtype=F16)
    assert y[45].isnan().all() and not y[50].isfinite().any() and y[40:340, 7].isnan().all()
    y[45], y[50], y[40:340, 7] = 0, 0, 0
    assert y.isfinite().all()
    ref.check_product(y[:40], x.view(torch.uint8)[:40].view(ref.F8), xs[:40], q[0], s[0])
    ref.check_product(y[340:], x.view(torch.uint8)[340:].view(ref.F8), xs[340:], q[2], s[2])


@pytest.mark.parametrize("bt", KERNELS)
def test_many_segments_and_long_sums(dev, bt):
    lens = torch.bincount(torch.randint(60, (9000,), generator=torch.Generator().manual_seed(bt)), minlength=60).tolist()
    q, s = ref.weights(dev, (60, 384, 2048), 1)
    x, xs = ref.activations(dev, 3000, 2048, 2)
    rows = torch.randint(3000, (9000,), device=dev, generator=ref.gen(dev, 3)).int()
    off = starts(dev, lens)
    w = ops.tile_f8(q, s)
    y = ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=rows, dtype=F16)
    c = off.tolist()
    for i in range(60):
        at = rows[c[i]:c[i + 1]].long()
        ref.check_product(y[c[i]:c[i + 1]], rows_of(x, at), xs[at], q[i], s[i], f"segment {i}")
    assert torch.equal(ops.matmul_f8_grouped_choice(w, x, xs, off, bt, rows=rows, dtype=F16), y)


def test_far_rows_by_index(dev):
    """rows by index more than 2^32 bytes from the first: not by the kernel with 32-bit offsets, whatever the sizes; in order by any"""
    t, n, k, lens = 260, 2048, 2048, [2560, 2560]
    q, s = ref.weights(dev, (2, n, k), 3)
    w = ops.tile_f8(q, s)
    x, xs = ref.activations(dev, t, k, 4)
    far = torch.empty(t << 24, dtype=torch.uint8, device=dev).view(ref.F8).as_strided((t, k), ((1 << 24) - 16, 1))
    far.view(torch.uint8).copy_(x.view(torch.uint8))
    xs_far = torch.empty(t << 22, device=dev).as_strided(xs.shape, ((1 << 22) - 1, 1))
    xs_far.copy_(xs)
    rows = torch.arange(sum(lens), dtype=torch.int32, device=dev) % t
    off = starts(dev, lens)
    for one, scales in ((far, xs), (x, xs_far), (far, xs_far)):
        with pytest.raises(ValueError, match="no blocks of 256"):
            ops.matmul_f8_grouped_choice(w, one, scales, off, 256, rows=rows)
        y = ops.matmul_f8_grouped(w, one, scales, off, rows=rows, dtype=F16)
        for i in range(2):
            at = rows[2560 * i:2560 * (i + 1)].long()
            ref.check_product(y[2560 * i:2560 * (i + 1)], rows_of(x, at), xs[at], q[i], s[i])
    off = starts(dev, [100, 160])
    want = ops.matmul_f8_grouped_choice(w, x, xs, off, 256)
    assert torch.equal(ops.matmul_f8_grouped_choice(w, far, xs_far, off, 256), want)
    ref.check_product(want[:100], rows_of(x, slice(0, 100)), xs[:100], q[0], s[0])


@pytest.mark.parametrize("bt", KERNELS)
def test_captured(dev, bt):
    q, s = ref.weights(dev, (3, 300, 1040), 5)
    x, xs = ref.activations(dev, 700, 1040, 6)
    w, off = ops.tile_f8(q, s), starts(dev, [300, 0, 400])
    xs = xs.contiguous()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out = ops.matmul_f8_grouped_choice(w, x, xs, off, bt)
    for i in range(3):
        xs.mul_(1.25)
        off[1] = 100 * (i + 1)
        off[2] = 100 * (i + 1)
        want = ops.matmul_f8_grouped_choice(w, x, xs, off, bt)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
