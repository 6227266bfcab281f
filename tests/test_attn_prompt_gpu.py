"""Causal attention of packed prompts against the formula in 64 bits (bounds: attention_ref.py)."""
import pytest
import torch

import attention_ref as ref
from qengine_amd import ops

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def starts(lens, dev, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=dev)


def inputs(dev, lens, heads, kv, d, dtype, seed, tail=0, first=0, spread=1.0):
    """q, k, v as views of one fused product"""
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    t = first + sum(lens) + tail
    x = (torch.randn(t, (heads + 2 * kv) * d, device=dev, generator=g) * spread).to(dtype)
    q, k, v = x.split([heads * d, kv * d, kv * d], 1)
    return q.view(t, heads, d), k.view(t, kv, d), v.view(t, kv, d), starts(lens, dev, first)


def compare(q, k, v, cu, out, lse, scale=None):
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    c = cu.tolist()
    for b, (a, e) in enumerate(zip(c[:-1], c[1:])):
        for r in range(a, e, 1024):
            z = min(e, r + 1024)
            seen = torch.arange(a, z, device=q.device)[None] <= torch.arange(r, z, device=q.device)[:, None]
            for h in range(heads):
                m = h // (heads // kv)
                want = ref.rows(q[r:z, h], k[a:z, m], v[a:z, m], seen, d ** -0.5 if scale is None else scale)
                ref.check(out[r:z, h], None if lse is None else lse[r:z, h], *want, what=f"sequence {b} rows {r - a}.. head {h}")


LENS = [[1], [2, 1], [0, 5, 0, 33, 64, 65], [127, 1, 128, 129, 0], [63, 300, 31, 32], [257]]


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_prompt(dev, lens, d, dtype):
    q, k, v, cu = inputs(dev, lens, 4, 2, d, dtype, seed=len(lens) + d)
    out, lse = ops.attn_prompt(q, k, v, cu, lse=True)
    compare(q, k, v, cu, out, lse)


@pytest.mark.parametrize("heads,kv", [(1, 1), (10, 2), (7, 7), (8, 1), (21, 3), (40, 8)])
def test_head_layouts(dev, heads, kv):
    q, k, v, cu = inputs(dev, [70, 0, 150], heads, kv, 128, BF, seed=heads)
    compare(q, k, v, cu, *ops.attn_prompt(q, k, v, cu, lse=True))


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF), (256, BF)])
def test_long(dev, d, dtype):
    q, k, v, cu = inputs(dev, [3001, 1], 2, 1, d, dtype, seed=5)
    compare(q, k, v, cu, *ops.attn_prompt(q, k, v, cu, lse=True))


# shapes of every tile choice: blocks of 128 rows in steps of 32 and 64 keys, blocks of 64 rows in groups
@pytest.mark.parametrize("lens,heads,kv,d,dtype", [
    ([1700, 1, 255, 64], 40, 8, 128, BF), ([700], 40, 8, 128, F16), ([2000], 8, 1, 128, BF), ([333, 129], 40, 8, 128, BF),
    ([3000], 32, 4, 64, BF), ([500, 31, 33, 257], 64, 8, 64, F16), ([2000], 16, 2, 64, BF),
    ([2100, 40], 32, 2, 256, BF), ([1000], 16, 2, 256, F16), ([2000], 16, 2, 256, BF)])
def test_tile_choices(dev, lens, heads, kv, d, dtype):
    q, k, v, cu = inputs(dev, lens, heads, kv, d, dtype, seed=sum(lens))
    group = heads // kv
    out, lse = ops.attn_prompt(q, k, v, cu, lse=True)
    for h in (0, heads // 2, heads - 1):
        m = h // group
        compare(q[:, h:h + 1], k[:, m:m + 1], v[:, m:m + 1], cu, out[:, h:h + 1], lse[:, h:h + 1])
    assert torch.equal(out, ops.attn_prompt(q, k, v, cu))


@pytest.mark.parametrize("nseq", [63, 64, 65, 300])
def test_many_sequences(dev, nseq):
    lens = [(i * 37) % 90 if i % 7 else 0 for i in range(nseq)]
    lens[nseq // 2] = 400
    q, k, v, cu = inputs(dev, lens, 2, 1, 64, BF, seed=nseq)
    compare(q, k, v, cu, ops.attn_prompt(q, k, v, cu), None)


def test_steep_scores_and_scale(dev):
    """scores that grow along the keys (the running maximum moves at every step), and large ones"""
    q, k, v, cu = inputs(dev, [500], 2, 1, 128, BF, seed=3, spread=2.0)
    k[:, 0] *= torch.linspace(0.1, 3, 500, device=dev)[:, None].to(BF)
    compare(q, k, v, cu, *ops.attn_prompt(q, k, v, cu, lse=True))
    compare(q, k, v, cu, *ops.attn_prompt(q, k, v, cu, scale=0.5, lse=True), scale=0.5)


def test_rows_outside_sequences_stay(dev):
    q, k, v, cu = inputs(dev, [40, 90], 4, 2, 128, BF, seed=4, tail=70, first=5)
    q[:5], q[135:], k[:5], k[135:], v[:5], v[135:] = (float("nan"),) * 6
    out = torch.full_like(q, 7.0)
    got = ops.attn_prompt(q, k, v, cu, out=out)
    assert got is out and (out[:5] == 7).all() and (out[135:] == 7).all()
    compare(q, k, v, cu, out, None)


def test_strides_of_out_and_heads(dev):
    """head-major inputs, an output inside a wider buffer"""
    q, k, v, cu = inputs(dev, [77, 20], 4, 2, 64, F16, seed=6)
    want = ops.attn_prompt(q, k, v, cu)
    hm = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    buf = torch.full((97, 4, 72), 3.0, dtype=F16, device=dev)
    ops.attn_prompt(*hm, cu, out=buf[:, :, :64])
    assert torch.equal(buf[:, :, :64], want) and (buf[:, :, 64:] == 3).all()


@pytest.mark.parametrize("heads", [2, 160])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_later_keys_that_are_not_finite(dev, bad, d, heads):
    """a row is not touched by what later keys and values hold; the rows that see them get what the formula says"""
    q, k, v, cu = inputs(dev, [150, 200], heads, 1, d, BF, seed=8)
    v[100, 0, 3] = bad          # rows 100.. of the first sequence see it
    k[150 + 130, 0, 5] = float("nan")
    out = ops.attn_prompt(q, k, v, cu)
    clean = v.clone()
    clean[100, 0, 3] = 0
    seen = torch.ones(100, 100, dtype=torch.bool, device=dev).tril()
    for h in (0, heads - 1):
        ref.check(out[:100, h], None, *ref.rows(q[:100, h], k[:100, 0], v[:100, 0], seen, d ** -0.5))
        seen2 = torch.ones(130, 130, dtype=torch.bool, device=dev).tril()
        ref.check(out[150:280, h], None, *ref.rows(q[150:280, h], k[150:280, 0], v[150:280, 0], seen2, d ** -0.5))
        assert torch.isnan(out[280:, h]).all()
        col = out[100:150, h, 3].float()
        assert torch.isnan(col).all() if bad != bad else (col == bad).all()
        full = torch.ones(150, 150, dtype=torch.bool, device=dev).tril()[100:]
        o, _, ob, _ = ref.rows(q[100:150, h], k[:150, 0], clean[:150, 0], full, d ** -0.5)
        rest = [i for i in range(d) if i != 3]
        ref.check(out[100:150, h][:, rest], None, o[:, rest], None, ob[:, rest], None)


def test_starts_out_of_range(dev):
    """starts that leave the tensors (a caller's mistake): nothing outside is touched, sequences inside are served"""
    q, k, v, cu = inputs(dev, [30, 34], 2, 1, 64, BF, seed=9)
    out = torch.full_like(q, 7.0)
    ops.attn_prompt(q, k, v, torch.tensor([-9, 30, 64, 5000, 20, 10], dtype=torch.int32, device=dev), out=out)
    compare(q, k, v, cu, out, None)


def test_nothing_to_do(dev):
    q, k, v, cu = inputs(dev, [0, 0], 2, 1, 64, BF, seed=9)
    assert ops.attn_prompt(q, k, v, cu).shape == (0, 2, 64)
    q, k, v, _ = inputs(dev, [8], 2, 1, 64, BF, seed=9)
    out = torch.full_like(q, 7.0)
    ops.attn_prompt(q, k, v, torch.zeros(1, dtype=torch.int32, device=dev), out=out)
    ops.attn_prompt(q, k, v, torch.zeros(4, dtype=torch.int32, device=dev), out=out)
    assert (out == 7).all()


def test_same_bits_streams_and_graph(dev):
    q, k, v, cu = inputs(dev, [200, 90, 1, 40], 8, 2, 128, BF, seed=10)
    want = ops.attn_prompt(q, k, v, cu)
    assert torch.equal(want, ops.attn_prompt(q, k, v, cu))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attn_prompt(q, k, v, cu)
    side.synchronize()
    assert torch.equal(want, other)
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_prompt(q, k, v, cu, out=out)
    for seed in (11, 12, 13):
        x = inputs(dev, [200, 90, 1, 40], 8, 2, 128, BF, seed=seed)
        q.copy_(x[0]), k.copy_(x[1]), v.copy_(x[2])
        cu.copy_(starts([30 * seed - 300, 331 - 30 * seed + 300, 0, 0], dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.attn_prompt(q, k, v, cu)), seed
