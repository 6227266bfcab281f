"""Products of 8-bit weights and activations against their formula in 64 bits (bounds: f8_ref.py)."""
import threading

import pytest
import torch

import f8_ref as ref
from qengine_amd import call, ops

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def linear(dev, t, n, k, dtype=F16, pad=0):
    x, xs = ref.activations(dev, t, k, t + 1, pad)
    q, s = ref.weights(dev, (n, k), n + k)
    y = ops.matmul_f8(ops.tile_f8(q, s), x, xs, dtype=dtype)
    assert y.dtype == dtype and y.shape == (t, n)
    ref.check_product(y, x, xs, q, s, f"{t} x {n} x {k}")


# rows around every bound between kernels and tiles
ROWS = [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 250, 256, 257, 500, 1023, 1025, 1300]


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("n,k", [(640, 1024), (257, 400)])
def test_rows(dev, t, n, k):
    linear(dev, t, n, k)


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("n,k", [(640, 1024), (257, 400)])
def test_whole_numbers(dev, t, n, k):
    """whole numbers up to 8 and scales that are powers of two: every product and sum is exact, so the output is the sum rounded once"""
    g = ref.gen(dev, t)
    x = torch.randint(-8, 9, (t, k), device=dev, generator=g).float().to(ref.F8)
    q = torch.randint(-8, 9, (n, k), device=dev, generator=g).float().to(ref.F8)
    xs = torch.exp2(torch.randint(-3, 1, (t, -(-k // 128)), device=dev, generator=g).float())
    s = torch.exp2(torch.randint(-3, 1, (-(-n // 128), -(-k // 128)), device=dev, generator=g).float())
    want = ref.product(x, xs, q, s)[0]  # below 2^16 in steps of 2^-6
    for dtype in (BF, F16):
        assert torch.equal(ops.matmul_f8(ops.tile_f8(q, s), x, xs, dtype=dtype), want.to(dtype))
    off = torch.tensor([0, t // 3, t // 3, t], dtype=torch.int32, device=dev)
    w = ops.tile_f8(torch.stack([q.view(torch.uint8)] * 3).view(ref.F8), torch.stack([s, s * 4, s * 2]))
    want[t // 3:] *= 2
    assert torch.equal(ops.matmul_f8_grouped(w, x, xs, off, dtype=F16), want.to(F16))


BLOCKS = [(16, 0)] + [(bt, bw) for bt in (32, 64, 128) for bw in (64, 128, 192)] + [(256, 256)]


@pytest.mark.parametrize("parts", [1, 2, 3, 7])
@pytest.mark.parametrize("bt,bw", BLOCKS)
def test_blocks(dev, bt, bw, parts):
    """every shape of a block and number of K ranges, whole and ragged tiles, K with a short block"""
    for t, n, k in [(bt, bw or 64, 896), (bt + 1, 2 * bw + 130, 1040), (max(bt // 2 - 3, 1), 97, 912), (2 * bt + 9, 3 * bw + 16, 2000)]:
        x, xs = ref.activations(dev, t, k, t + 1, 16)
        q, s = ref.weights(dev, (n, k), n + k)
        ref.check_product(ops.matmul_f8_choice(ops.tile_f8(q, s), x, xs, bt, bw, parts), x, xs, q, s, f"{t} x {n} x {k}")
        g = ref.gen(dev, t)
        x = torch.randint(-8, 9, (t, k), device=dev, generator=g).float().to(ref.F8)
        q = torch.randint(-8, 9, (n, k), device=dev, generator=g).float().to(ref.F8)
        xs = torch.exp2(torch.randint(-3, 1, (-(-k // 128), t), device=dev, generator=g).float()).t()
        s = torch.exp2(torch.randint(-3, 1, (-(-n // 128), -(-k // 128)), device=dev, generator=g).float())
        want = ref.product(x, xs, q, s)[0]
        assert torch.equal(ops.matmul_f8_choice(ops.tile_f8(q, s), x, xs, bt, bw, parts, dtype=F16), want.to(F16)), f"{t} x {n} x {k}"


# odd ends of both sides, one block, one column, deep sums
@pytest.mark.parametrize("t", [1, 20, 50, 200, 1100])
@pytest.mark.parametrize("n,k", [(1, 16), (1, 128), (15, 144), (16, 128), (17, 112), (127, 256), (129, 272), (130, 4096), (384, 2064), (1000, 528)])
def test_sizes(dev, t, n, k):
    linear(dev, t, n, k, pad=32)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("t", [1, 40, 300, 1500])
def test_types(dev, t, dtype):
    linear(dev, t, 512, 640, dtype)
    linear(dev, t, 509, 640, dtype)


@pytest.mark.parametrize("t,n,k", [(1, 5120, 17408), (1, 34816, 5120), (24, 5120, 17408), (48, 34816, 5120), (100, 5120, 17408), (128, 34816, 5120),
                                   (1000, 5120, 17408), (2100, 17408, 5120)])
def test_large(dev, t, n, k):
    linear(dev, t, n, k, BF)


@pytest.mark.parametrize("t", [3, 40, 200, 1100])
def test_strides(dev, t):
    """rows apart, scales row-major, an output with rows apart and not aligned"""
    q, s = ref.weights(dev, (260, 640), 3)
    w = ops.tile_f8(q, s)
    x, xs = ref.activations(dev, t, 640, 4, pad=48)
    want = ops.matmul_f8(w, x.contiguous(), xs, dtype=BF)
    for out, more in [(BF, 4), (BF, 3), (F16, 8), (F16, 9)]:
        room = torch.full((t, 260 + more), 7.0, dtype=out, device=dev)
        assert ops.matmul_f8(w, x, xs.contiguous(), y=room[:, :260]).data_ptr() == room.data_ptr()
        assert (room[:, 260:] == 7).all()
        ref.check_product(room[:, :260], x, xs, q, s)
        if out == BF:
            assert torch.equal(room[:, :260], want)


@pytest.mark.parametrize("t", [4, 40, 200, 1100])
def test_values_stay_in_their_rows(dev, t):
    """a NaN or an infinite scale spoils its row or its columns and nothing else"""
    q, s = ref.weights(dev, (300, 528), 5)
    x, xs = ref.activations(dev, t, 528, 6)
    x, xs = x.contiguous(), xs.clone()
    x.view(torch.uint8)[1, 520] = 0x7F
    xs[2, 4] = float("inf")
    q.view(torch.uint8)[7, 3] = 0xFF
    y = ops.matmul_f8(ops.tile_f8(q, s), x, xs, dtype=F16)
    rows = [i for i in range(t) if i not in (1, 2)]
    cols = [i for i in range(300) if i != 7]
    assert y[1].isnan().all() and not y[2].isfinite().any() and y[:, 7].isnan().all()
    keep = q.clone()
    keep.view(torch.uint8)[7, 3] = 0
    want, off = ref.product(x.view(torch.uint8)[rows].view(ref.F8), xs[rows], keep, s)
    ref.within(y[rows][:, cols], want[:, cols], (off + ref.half(F16, want.abs() + off))[:, cols])


def test_tile_strides(dev):
    q, s = ref.weights(dev, (3, 140, 272), 8)
    x, xs = ref.activations(dev, 5, 272, 9)
    off = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=dev)
    want = ops.matmul_f8_grouped(ops.tile_f8(q, s), x, xs, off)
    room = torch.zeros(3, 140, 304, device=dev).to(ref.F8)
    room[:, :, :272] = q
    for other in (room[:, :, :272], q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(ops.matmul_f8_grouped(ops.tile_f8(other, s), x, xs, off), want)


def grouped(dev, lens, n, k, dtype=F16, gather=None, first=0, tail=0, seed=0):
    e, r = len(lens), first + sum(lens) + tail
    q, s = ref.weights(dev, (e, n, k), seed + 1)
    t = gather or r
    x, xs = ref.activations(dev, t, k, seed + 2, pad=16)
    off = torch.tensor([first + sum(lens[:i]) for i in range(e + 1)], dtype=torch.int32, device=dev)
    rows = torch.randint(t, (r,), device=dev, generator=ref.gen(dev, seed)).int() if gather else None
    y = torch.full((r, n), 7.0, dtype=dtype, device=dev)
    assert ops.matmul_f8_grouped(ops.tile_f8(q, s), x, xs, off, rows=rows, y=y) is y
    assert (y[:first] == 7).all() and (y[r - tail:] == 7).all()
    c = off.tolist()
    for i in range(e):
        if lens[i]:
            at = torch.arange(c[i], c[i + 1], device=dev) if rows is None else rows[c[i]:c[i + 1]].long()
            ref.check_product(y[c[i]:c[i + 1]], x.view(torch.uint8)[at].view(ref.F8), xs[at], q[i], s[i], f"segment {i} of {lens[i]}")


LENS = [[1], [0, 3, 0], [700, 0, 513, 256], [16, 17, 1, 15, 0, 33], [64, 65, 128, 129, 0, 200], [0] * 30 + [5] + [0] * 33, [300], [40] * 20, [0, 0]]


@pytest.mark.parametrize("lens", LENS, ids=lambda v: str(v)[:24])
@pytest.mark.parametrize("n,k", [(640, 512), (65, 208)])
@pytest.mark.parametrize("gather", [None, 9])
def test_grouped(dev, lens, n, k, gather):
    grouped(dev, lens, n, k, gather=gather, first=2, tail=3)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_grouped_types(dev, dtype):
    grouped(dev, [3, 0, 20, 100], 257, 384, dtype)


@pytest.mark.parametrize("experts,tokens", [(512, 160), (512, 3000), (512, 7000), (1024, 1024), (60, 2000), (30, 2500), (7, 5000)])
def test_grouped_many(dev, experts, tokens):
    g = torch.Generator().manual_seed(experts)
    lens = torch.bincount(torch.randint(experts, (tokens,), generator=g), minlength=experts).tolist()
    grouped(dev, lens, 128, 256, gather=tokens // 3)


def test_grouped_bad_indexes(dev):
    """rows outside x give zeros; segments that do not ascend or leave y write nothing outside"""
    q, s = ref.weights(dev, (4, 96, 128), 1)
    x, xs = ref.activations(dev, 6, 128, 2)
    w = ops.tile_f8(q, s)
    rows = torch.tensor([0, -1, 6, 5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)
    off = torch.tensor([0, 6, 6, 6, 6], dtype=torch.int32, device=dev)
    y = ops.matmul_f8_grouped(w, x, xs, off, rows=rows, dtype=F16)
    assert (y[[1, 2, 4, 5]] == 0).all() and (y[[0, 3]] != 0).any(1).all()
    for bad in ([3, 1, 9, 2, 4], [-5, 2, 2, 100, 3], [2 ** 31 - 1, 0, 0, 0, -2 ** 31]):
        room = torch.full((20, 96), 7.0, dtype=BF, device=dev)
        off = torch.tensor(bad, dtype=torch.int32, device=dev)
        ops.matmul_f8_grouped(w, x, xs, off, y=room[7:13])
        assert (room[:7] == 7).all() and (room[13:] == 7).all()


@pytest.mark.parametrize("lens,n,k", [([5, 0, 9], 97, 272), ([30, 100, 1], 640, 512), ([300, 0, 260], 640, 512), ([2100, 900], 1024, 400)])
def test_grouped_bad_indexes_by_every_kernel(dev, lens, n, k):
    """as row 0, but zeros"""
    e, r, t = len(lens), sum(lens), 50
    q, s = ref.weights(dev, (e, n, k), 1)
    x, xs = ref.activations(dev, t, k, 2)
    w = ops.tile_f8(q, s)
    off = torch.tensor([sum(lens[:i]) for i in range(e + 1)], dtype=torch.int32, device=dev)
    g = ref.gen(dev, r)
    rows = torch.randint(t, (r,), device=dev, generator=g).int()
    bad = torch.rand(r, device=dev, generator=g) < 0.3
    bad[0] = bad[-1] = True
    far = torch.tensor([-1, t, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)[torch.arange(r, device=dev) % 4]
    want = ops.matmul_f8_grouped(w, x, xs, off, rows=torch.where(bad, 0, rows))
    y = ops.matmul_f8_grouped(w, x, xs, off, rows=torch.where(bad, far, rows))
    assert torch.equal(y, torch.where(bad[:, None], 0, want))


@pytest.mark.parametrize("t", [3, 40, 300])
def test_far_rows(dev, t):
    """rows and scales as far apart as a call takes, so that offsets pass 32 bits"""
    n, k = 530, 400
    q, s = ref.weights(dev, (n, k), 3)
    w, one = ops.tile_f8(q, s), ops.tile_f8(q[None], s[None])
    x, xs = ref.activations(dev, t, k, 4)
    want = ops.matmul_f8(w, x, xs)
    far = torch.empty(t << 24, dtype=torch.uint8, device=dev).view(ref.F8).as_strided((t, k), ((1 << 24) - 16, 1))
    far.view(torch.uint8).copy_(x.view(torch.uint8))
    xs_far = torch.empty(t << 22, device=dev).as_strided(xs.shape, ((1 << 22) - 1, 1))
    xs_far.copy_(xs)
    assert torch.equal(ops.matmul_f8(w, far, xs_far), want)
    off = torch.tensor([0, t], dtype=torch.int32, device=dev)
    rows = torch.arange(t - 1, -1, -1, dtype=torch.int32, device=dev)
    back = rows.long()
    ref.check_product(ops.matmul_f8_grouped(one, far, xs_far, off, dtype=F16), x, xs, q, s)
    ref.check_product(ops.matmul_f8_grouped(one, far, xs_far, off, rows=rows, dtype=F16), x.view(torch.uint8)[back].view(ref.F8), xs[back], q, s)


def test_large_outputs_and_weights(dev):
    """y and the experts' weights beyond 2^32 bytes: what lies last"""
    t, n, k = 17000, 131072, 128
    q, s = ref.weights(dev, (n, k), 5)
    x, xs = ref.activations(dev, t, k, 6)
    y = ops.matmul_f8(ops.tile_f8(q, s), x, xs)
    last, cols = slice(t - 300, t), slice(n - 512, n)
    ref.check_product(y[last, cols], x.view(torch.uint8)[last].view(ref.F8), xs[last], q.view(torch.uint8)[cols].view(ref.F8), s[-4:], "last")
    del y
    e, n, k = 1024, 2048, 2560
    q, s = ref.weights(dev, (2, n, k), 7)
    many = torch.zeros(e, n, k, dtype=torch.uint8, device=dev)
    many[0], many[-1] = q.view(torch.uint8)[0], q.view(torch.uint8)[1]
    scales = torch.ones(e, *s.shape[1:], device=dev)
    scales[0], scales[-1] = s[0], s[1]
    w = ops.tile_f8(many.view(ref.F8), scales)
    del many
    for lens in ([3, 2], [5000, 4000]):
        off = torch.full((e + 1,), lens[0], dtype=torch.int32, device=dev)
        off[0], off[-1] = 0, sum(lens)
        x, xs = ref.activations(dev, sum(lens), k, 8)
        y = ops.matmul_f8_grouped(w, x, xs, off, dtype=F16)
        tail = slice(sum(lens) - lens[1], sum(lens))
        for rows, i in ((slice(0, lens[0]), 0), (tail, 1)):
            ref.check_product(y[rows], x.view(torch.uint8)[rows].view(ref.F8), xs[rows], q[i], s[i], f"{lens} {i}")


def test_no_rows(dev):
    q, s = ref.weights(dev, (2, 32, 128), 1)
    x, xs = ref.activations(dev, 0, 128, 2)
    assert ops.matmul_f8(ops.tile_f8(q[0], s[0]), x, xs).shape == (0, 32)
    off = torch.zeros(3, dtype=torch.int32, device=dev)
    assert ops.matmul_f8_grouped(ops.tile_f8(q, s), x, xs, off).shape == (0, 32)
    rows = torch.zeros(4, dtype=torch.int32, device=dev)  # rows, but none to take
    off = torch.tensor([0, 1, 4], dtype=torch.int32, device=dev)
    assert (ops.matmul_f8_grouped(ops.tile_f8(q, s), x, xs, off, rows=rows) == 0).all()


@pytest.mark.parametrize("t", [1, 20, 60, 300])
def test_same_bits_again(dev, t):
    q, s = ref.weights(dev, (512, 2048), 1)
    x, xs = ref.activations(dev, t, 2048, 2)
    w = ops.tile_f8(q, s)
    first = ops.matmul_f8(w, x, xs, dtype=F16)
    for _ in range(5):
        assert torch.equal(ops.matmul_f8(w, x, xs, dtype=F16), first)


def mlp(x, h, norm, w1, w2):
    q, s = ops.rms_norm(x, norm, res=h, f8=True)
    return ops.matmul_f8(w2, *ops.silu_mul_f8(ops.matmul_f8(w1, q, s)))


def experts(x, logits, w1, w2, topk, add):
    """route -> segment -> first product, rows gathered -> activation -> second -> back into tokens"""
    sel, w = ops.moe_route(logits, topk)
    seg = ops.moe_segment(sel, w, logits.shape[1], 64)
    q, s = ops.quant_f8(x)
    g = ops.matmul_f8_grouped(w1, q, s, seg["off"], rows=seg["slot_tok"])
    y = ops.matmul_f8_grouped(w2, *ops.silu_mul_f8(g), seg["off"])
    return ops.moe_combine(y, seg["inv"], w, add=add)


def layers(dev, t, hidden, inter, n_experts, seed=0):
    g = ref.gen(dev, seed)

    def mats(*lead, n, k):
        w = torch.randn(*lead, n, k, device=dev, generator=g)
        return (w * 100).clamp(-448, 448).to(ref.F8), torch.full((*lead, -(-n // 128), -(-k // 128)), k ** -0.5 / 100, device=dev)

    x = torch.randn(t, hidden, device=dev, generator=g).to(BF)
    h = torch.randn(t, hidden, device=dev, generator=g).to(BF)
    return x, h, mats(n=2 * inter, k=hidden), mats(n=hidden, k=inter), mats(n_experts, n=2 * inter, k=hidden), mats(n_experts, n=hidden, k=inter)


@pytest.mark.parametrize("t", [1, 30, 200])
def test_mlp_and_experts_as_they_are_used(dev, t):
    """a block and an expert layer against the same steps in 64 bits, without the roundings to 8 bits between them: each of the
    two e4m3 roundings is off by at most 2^-4 of a value, so the result by 2^-3 of its norm and more; a misplaced
    group, row or expert by more than half of it"""
    hidden, inter, n_experts, topk = 512, 384, 16, 4
    x, h, m1, m2, e1, e2 = layers(dev, t, hidden, inter, n_experts)
    norm = torch.ones(hidden, device=dev)

    def product(v, m, e=None):
        q, s = m if e is None else (m[0][e], m[1][e])
        return v @ (q.double() * s.double()[..., :1, :1]).t().contiguous()

    stream = (x.float() + h.float()).to(BF)
    got = mlp(x, h, norm, ops.tile_f8(*m1), ops.tile_f8(*m2))
    assert torch.equal(h, stream)
    want = product(ref.silu_mul(product(ref.norm(stream, norm, 1e-6), m1)), m2)
    assert (got.double() - want).norm() <= 0.125 * want.norm()
    logits = torch.randn(t, n_experts, device=dev, generator=ref.gen(dev, 9))
    got = experts(x, logits, ops.tile_f8(*e1), ops.tile_f8(*e2), topk, h)
    top, sel = logits.double().topk(topk)
    w = torch.softmax(top, -1)
    want = stream.double()
    for i in range(t):
        for j in range(topk):
            e = int(sel[i, j])
            want[i] += w[i, j] * product(ref.silu_mul(product(x[i:i + 1].double(), e1, e)), e2, e)[0]
    assert (got.double() - want).norm() <= 0.125 * (want - stream.double()).norm() + 2 ** -8 * want.norm()


@pytest.mark.parametrize("t", [1, 12, 200])
def test_captured(dev, t):
    """a layer in a graph, replayed on new inputs beside eager calls"""
    hidden, inter, n_experts, topk = 512, 384, 16, 4
    x, h, m1, m2, e1, e2 = layers(dev, t, hidden, inter, n_experts, 3)
    norm = torch.ones(hidden, device=dev)
    w = [ops.tile_f8(*m) for m in (m1, m2, e1, e2)]
    logits = torch.randn(t, n_experts, device=dev)

    def step(x, h, logits):
        y = mlp(x, h, norm, w[0], w[1])
        return experts(y, logits, w[2], w[3], topk, h)

    side = torch.cuda.Stream()
    xs, hs, ls = x.clone(), h.clone(), logits.clone()
    with torch.cuda.stream(side):
        step(xs, hs.clone(), ls)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(xs, hs, ls)
    for i in range(4):
        g = ref.gen(dev, 50 + i)
        xs.copy_(torch.randn(xs.shape, device=dev, generator=g))
        hs.copy_(torch.randn(xs.shape, device=dev, generator=g))
        ls.copy_(torch.randn(ls.shape, device=dev, generator=g))
        h2 = hs.clone()
        want = step(xs, h2, ls)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(hs, h2)


def test_graphs_have_their_own_sums(dev):
    """products whose K is split use sums that their graph holds: two graphs of one stream replay beside each other and eager calls"""
    t, n, k = 300, 512, 8192
    q, s = ref.weights(dev, (n, k), 1)
    w = ops.tile_f8(q, s)
    ins = [ref.activations(dev, t, k, i) for i in range(3)]
    want = [ops.matmul_f8(w, *i) for i in ins]
    assert call("qe_workspace_count", 6) >= 1
    side = torch.cuda.Stream()
    before = call("qe_workspace_count", 6)
    graphs, outs = [], []
    for i in ins[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(ops.matmul_f8(w, *i))
        graphs.append(graph)
    assert call("qe_workspace_count", 6) == before + 2
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(8):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        eager = ops.matmul_f8(w, *ins[2])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])
    del graphs, graph
    torch.cuda.synchronize()
    assert call("qe_workspace_count", 6) == before


def test_threads_on_one_stream(dev):
    """split products of several host threads on the default stream do not mix their sums"""
    q, s = ref.weights(dev, (512, 8192), 1)
    w = ops.tile_f8(q, s)
    ins = [ref.activations(dev, 300, 8192, i) for i in range(4)]
    want = [ops.matmul_f8(w, *i) for i in ins]
    got = [[] for _ in ins]

    def work(i):
        for _ in range(25):
            got[i].append(ops.matmul_f8(w, *ins[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    torch.cuda.synchronize()
    for o, y in zip(got, want):
        assert len(o) == 25 and all(torch.equal(v, y) for v in o)


@pytest.mark.parametrize("t", [1, 60, 300, 1200])
def test_streams(dev, t):
    """two streams at once give what they give alone"""
    q, s = ref.weights(dev, (1024, 2048), 1)
    w = ops.tile_f8(q, s)
    ins = [ref.activations(dev, t, 2048, i) for i in range(2)]
    want = [ops.matmul_f8(w, *i, dtype=F16) for i in ins]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ins]
    got = [[], []]
    for _ in range(20):
        for st, i, o in zip(streams, ins, got):
            with torch.cuda.stream(st):
                o.append(ops.matmul_f8(w, *i, dtype=F16))
    torch.cuda.synchronize()
    for o, y in zip(got, want):
        assert all(torch.equal(v, y) for v in o)


def test_a_stream_allocates_its_sums_once(dev):
    """the first split product of a stream allocates what the largest may need: later ones of any size allocate nothing, and one
    whose sums need more runs unsplit"""
    k = 2048
    q, s = ref.weights(dev, (4096, k), 1)
    w = ops.tile_f8(q, s)
    x, xs = ref.activations(dev, 4096, k, 2)

    def product(t, n, bt, bw, parts):
        one = ops.F8(w.q[:n // 16 * (k // 128) * 2048], w.s[:n // 128], n, k)
        return ops.matmul_f8_choice(one, x[:t], xs[:t].t().contiguous().t(), bt, bw, parts)

    calls = [(40, 256, 64, 64, 2), (300, 512, 128, 128, 4), (1000, 1024, 256, 256, 4), (4096, 1024, 256, 256, 4), (1024, 4096, 256, 256, 4), (2048, 4096, 256, 256, 2)]
    too_large = [(4096, 4096, 256, 256, 2), (4096, 4096, 256, 256, 16), (4096, 4096, 128, 192, 2)]
    with torch.cuda.stream(torch.cuda.Stream()):
        whole = [product(*c[:4], 1) for c in calls + too_large]  # (torch's own blocks are there afterwards)
        got = [product(*c[:4], 1) for c in calls + too_large]
        del got
        got = [product(*calls[0])]
        torch.cuda.synchronize()
        count, free = call("qe_workspace_count", 6), torch.cuda.mem_get_info()[0]
        got += [product(*c) for c in calls[1:] + too_large]
        torch.cuda.synchronize()
        assert torch.cuda.mem_get_info()[0] == free and call("qe_workspace_count", 6) == count
    for c, a, b in zip(calls + too_large, got, whole):
        t, n = c[:2]
        ref.check_product(a, x[:t], xs[:t], q[:n], s[:n // 128], str(c))
        assert c not in too_large or torch.equal(a, b), c
