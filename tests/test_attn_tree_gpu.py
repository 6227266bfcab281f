"""Attention of drafted tokens over the paged cache against the formula in 64 bits (bounds: attention_ref.py)."""
import random

import pytest
import torch

import attention_ref as ref
from qengine_amd import call, lib, ops

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def ints(v, dev, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=dev)


def setup(dev, contexts, new, heads, kv, d, page, dtype, seed, stale=None, layers=1, order="nhd", tree=None):
    """-> (cache, q, seqs, cu, mask, Pages): a cache in use: pages in random order, slots in random order, what no sequence
    holds (and the rows behind a sequence's last) filled with `stale`"""
    rng = random.Random(seed)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    n = len(contexts)
    used = sum(-(-(c + x) // page) for c, x in zip(contexts, new))
    pages, slots = used + 5, n + 2
    width = max(-(-(c + x) // page) for c, x in zip(contexts, new)) + 1
    shape = (layers, pages, page, kv, d) if order == "nhd" else (layers, pages, kv, page, d)
    k, v = (torch.randn(shape, device=dev, generator=g).to(dtype) for _ in range(2))
    if order == "nhd":
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    free = rng.sample(range(pages), pages)
    place = rng.sample(range(slots), n)
    table, length, held, rf = [[-1] * width for _ in range(slots)], [0] * slots, [0] * slots, [0] * pages
    keep = torch.zeros(pages, page, dtype=torch.bool, device=dev)
    for s, c, x in zip(place, contexts, new):
        m = -(-(c + x) // page)
        for j in range(m):
            p = free.pop()
            table[s][j], rf[p] = p, 1
            keep[p, :min(page, c + x - j * page)] = True
        length[s], held[s] = c, m
    if stale is not None:
        gone = ~keep[None, :, None, :, None].expand(k.shape)
        k[gone], v[gone] = stale, stale
    cache = ops.KVCache(k, v, ints(table, dev), ints(length, dev), ints(held, dev), ints(rf, dev))
    q = torch.randn(sum(new), heads, d, device=dev, generator=g).to(dtype)
    cu = ints([sum(new[:i]) for i in range(n + 1)], dev)
    mask, words = None, None
    if tree:
        words = []
        for x in new:
            seen = []
            for i in range(x):
                if tree == "random":
                    seen.append(rng.getrandbits(64))  # also bits of tokens that do not exist, and rows without themselves
                elif tree == "none":
                    seen.append(0)
                else:
                    up = rng.randint(max(-1, i - 4), i - 1) if i else -1
                    seen.append((seen[up] if up >= 0 else 0) | 1 << i)
            words += seen
        mask = ints([w - (1 << 64) if w >> 63 else w for w in words], dev, torch.int64)
    return cache, q, ints(place, dev), cu, mask, words


def compare(cache, q, seqs, cu, words, out, lse, layer=0, scale=None, contexts=None):
    state = ref.Pages(cache)
    heads, kv, d = q.shape[1], cache.kv_heads, q.shape[2]
    c = cu.tolist()
    for b, s in enumerate(seqs.tolist()):
        a, e = c[b], c[b + 1]
        if e == a:
            continue
        n, x = state.length[s], e - a
        k, v = state.tokens(layer, s, n + x) if n + x else (None, None)
        seen = torch.ones(x, n + x, dtype=torch.bool)
        for i in range(x):
            w = words[a + i] if words else (1 << (i + 1)) - 1
            seen[i, n:] = torch.tensor([bool(w >> j & 1) for j in range(x)])
        for h in range(heads):
            m = h // (heads // kv)
            want = ref.rows(q[a:e, h], k[:, m], v[:, m], seen.to(q.device), d ** -0.5 if scale is None else scale)
            ref.check(out[a:e, h], None if lse is None else lse[a:e, h], *want, what=f"sequence {b} head {h}")


def attend(cache, q, seqs, cu, most, mask=None, **kw):
    return cache.attend(kw.pop("layer", 0), q, seqs, cu, most, mask=mask, **kw)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_decode(dev, page, d, dtype):
    """one token a sequence: contexts around the sizes of a page, a wave's 32 tokens and a unit, none, and long ones"""
    ctx = [0, 1, 14, 15, 16, 31, 32, 33, 63, 64, 127, 128, 129, 255, 700, 1500]
    c, q, seqs, cu, _, _ = setup(dev, ctx, [1] * len(ctx), 4, 2, d, page, dtype, seed=d + page, stale=float("nan"))
    compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, 1, lse=True))


@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 1), (16, 1), (17, 1), (33, 1), (40, 8), (6, 6), (128, 2)])
def test_head_layouts(dev, heads, kv):
    c, q, seqs, cu, _, _ = setup(dev, [100, 0, 333], [1, 2, 1], heads, kv, 128, 32, BF, seed=heads, stale=float("inf"))
    compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, 2, lse=True))


@pytest.mark.parametrize("tree", [None, "tree", "random", "none"])
@pytest.mark.parametrize("d,dtype", [(64, BF), (128, F16), (256, BF)])
def test_drafts(dev, d, dtype, tree):
    """chains and trees of up to 64 tokens, ragged, some sequences without rows; random masks hide tokens from themselves"""
    ctx, new = [0, 50, 7, 200, 31, 0, 1000, 64], [5, 64, 1, 33, 0, 64, 17, 2]
    c, q, seqs, cu, mask, words = setup(dev, ctx, new, 10, 2, d, 16, dtype, seed=d, stale=float("nan"), tree=tree)
    compare(c, q, seqs, cu, words, *attend(c, q, seqs, cu, 64, mask, lse=True))


def test_rows_that_see_nothing(dev):
    c, q, seqs, cu, mask, words = setup(dev, [0, 0, 40], [3, 1, 2], 4, 1, 64, 16, BF, seed=2, tree="none")
    out, lse = attend(c, q, seqs, cu, 3, mask, lse=True)
    assert (out[:4] == 0).all() and (lse[:4] == float("-inf")).all()
    compare(c, q, seqs, cu, words, out, lse)


@pytest.mark.parametrize("order", ["nhd", "hnd"])
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
def test_pages_and_orders(dev, page, order):
    c, q, seqs, cu, mask, words = setup(dev, [900, 15, 2049, 100], [4, 9, 1, 16], 8, 2, 128, page, BF, seed=page, tree="tree",
                                        layers=2, order=order, stale=float("-inf"))
    compare(c, q, seqs, cu, words, *attend(c, q, seqs, cu, 16, mask, lse=True, layer=1), layer=1)


@pytest.mark.parametrize("d,heads,kv,new", [(128, 8, 2, 1), (256, 8, 1, 5), (64, 16, 1, 64), (128, 5, 1, 40)])
def test_long_contexts(dev, d, heads, kv, new):
    """one sequence over all compute units, and next to short ones: sums in many parts"""
    c, q, seqs, cu, mask, words = setup(dev, [70001], [new], heads, kv, d, 64, BF, seed=d)
    compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, new, lse=True))
    c, q, seqs, cu, mask, words = setup(dev, [20000, 3, 500, 9000], [new, 1, new, 1], heads, kv, d, 64, F16, seed=d)
    compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, new, lse=True))


def test_large_batches(dev):
    """more sequences than threads that count them"""
    ctx = [(i * 53) % 150 for i in range(700)]
    c, q, seqs, cu, _, _ = setup(dev, ctx, [1 if i % 5 else 0 for i in range(700)], 2, 1, 64, 16, BF, seed=3)
    compare(c, q, seqs, cu, None, attend(c, q, seqs, cu, 1), None)


def test_offsets_past_32_bits(dev):
    """pools of more than 2^32 bytes (and elements), the sequence's pages at their end"""
    pages, page = 35000, 64
    k = torch.zeros(1, pages, 2, page, 512, dtype=BF, device=dev)[..., :128]
    v = torch.zeros(1, pages, 2, page, 512, dtype=BF, device=dev)[..., :128]
    assert k.stride(1) * pages > 2 ** 31
    table = [[-1] * 4, [pages - 1, pages - 3, 1, -1]]
    rf = torch.zeros(pages, dtype=torch.int32, device=dev)
    g = torch.Generator(device=dev)
    g.manual_seed(1)
    for p in (pages - 1, pages - 3, 1):
        k[:, p], v[:, p] = (torch.randn(1, 2, page, 128, device=dev, generator=g).to(BF) for _ in range(2))
        rf[p] = 1
    c = ops.KVCache(k, v, ints(table, dev), ints([0, 150], dev), ints([0, 3], dev), rf)
    q = torch.randn(3, 4, 128, device=dev, generator=g).to(BF)
    seqs, cu = ints([1], dev), ints([0, 3], dev)
    out, lse = attend(c, q, seqs, cu, 3, lse=True)
    pg = torch.tensor(table[1][:3], device=dev)
    kk, vv = (x[0, pg].transpose(1, 2).reshape(-1, 2, 128)[:153] for x in (k, v))
    seen = torch.ones(3, 153, dtype=torch.bool, device=dev).tril(150)
    for h in range(4):
        ref.check(out[:, h], lse[:, h], *ref.rows(q[:, h], kk[:, h // 2], vv[:, h // 2], seen, 128 ** -0.5))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("new,context", [(20, 45), (7, 45), (7, 5000), (20, 5000), (64, 900)])
def test_drafts_that_are_not_finite(dev, bad, d, new, context):
    """a drafted value that some rows see: theirs is what the formula says, the others' as if it were not there"""
    c, q, seqs, cu, mask, words = setup(dev, [context], [new], 2, 1, d, 16, BF, seed=7, tree="tree")
    s, col = seqs.item(), 3
    state = ref.Pages(c)
    pg, off = state.place(s, context + 2)
    c.v[0, pg, 0, off, col] = bad
    out = attend(c, q, seqs, cu, new, mask)
    k, v = state.tokens(0, s, context + new)
    sees = [i for i in range(new) if words[i] >> 2 & 1]
    others = [i for i in range(new) if i not in sees]
    assert sees and others
    seen = torch.ones(new, context + new, dtype=torch.bool)
    for i in range(new):
        seen[i, context:] = torch.tensor([bool(words[i] >> j & 1) for j in range(new)])
    clean = v.clone()
    clean[context + 2, 0, col] = 0
    rest = [i for i in range(d) if i != col]
    for h in range(2):
        o, _, ob, _ = ref.rows(q[:, h], k[:, 0], clean[:, 0], seen.to(dev), d ** -0.5)
        ref.check(out[others, h], None, o[others], None, ob[others], None)
        ref.check(out[sees, h][:, rest], None, o[sees][:, rest], None, ob[sees][:, rest], None)
        x = out[sees, h, col].float()
        assert torch.isnan(x).all() if bad != bad else (x == bad).all()


def test_steep_scores(dev):
    c, q, seqs, cu, _, _ = setup(dev, [2000, 300], [2, 1], 4, 2, 128, 32, BF, seed=9)
    q *= 4
    compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, 2, lse=True))
    compare(c, q, seqs, cu, None, *attend(c, q, seqs, cu, 2, lse=True, scale=1.5), scale=1.5)


def test_bad_slots_pages_and_starts(dev):
    """slots, pages and starts out of range (a caller's mistake): such rows see nothing or stay, the others are served"""
    c, q, seqs, cu, _, _ = setup(dev, [40, 100, 60], [1, 1, 1], 4, 2, 64, 16, BF, seed=11)
    want, wl = attend(c, q, seqs, cu, 1, lse=True)
    bad = seqs.clone()
    bad[1] = 99
    out, lse = attend(c, q, bad, cu, 1, lse=True)
    assert torch.equal(out[[0, 2]], want[[0, 2]]) and (out[1] == 0).all() and (lse[1] == float("-inf")).all()
    c.table[seqs[1], 2] = 1 << 30    # tokens 32 .. 47 of the second sequence are not there
    c.table[seqs[2], 3] = -7         # and 48 .. of the third
    out = attend(c, q, seqs, cu, 1)
    state = ref.Pages(c)
    for b, n, gone in ((1, 101, range(32, 48)), (2, 61, range(48, 61))):
        s = seqs[b].item()
        state.table[s] = [p if 0 <= p < c.pages else 0 for p in state.table[s]]
        k, v = state.tokens(0, s, n)
        seen = torch.tensor([[i not in gone for i in range(n)]], device=dev)
        for h in range(4):
            ref.check(out[b:b + 1, h], None, *ref.rows(q[b:b + 1, h], k[:, h // 2], v[:, h // 2], seen, 0.125))
    assert torch.equal(out[0], want[0])
    keep = torch.full_like(q, 7.0)
    attend(c, q, ints([0] * 5, dev), ints([-3, 0, 0, 70, 1, 9], dev), 1, out=keep)
    assert (keep[2:] == 7).all()  # the entries 0 .. 70 and 1 .. 9 name rows 0 and 1 (one each); row 2 is past `most` of both


def test_rows_outside_sequences_stay(dev):
    c, q, seqs, cu, _, _ = setup(dev, [40, 10], [3, 2], 4, 2, 128, 16, BF, seed=12)
    wide = torch.full((9, 4, 128), float("nan"), dtype=BF, device=dev)
    wide[2:7] = q
    out = torch.full_like(wide, 7.0)
    attend(c, wide, seqs, cu + 2, 3, out=out)
    assert (out[:2] == 7).all() and (out[7:] == 7).all()
    compare(c, q, seqs, cu, None, out[2:7], None)
    short = torch.full_like(q, 7.0)
    attend(c, q, seqs, cu, 2, out=short)  # most = 2: the third row of the first sequence stays
    assert (short[2] == 7).all() and torch.isfinite(short).all() and not (short[1] == 7).all()


@pytest.mark.parametrize("heads,d", [(4, 128), (10, 128), (10, 64), (64, 256), (64, 128)])
def test_without_parts(dev, heads, d):
    """a block takes whole rows where there is no memory for parts"""
    c, q, seqs, cu, mask, words = setup(dev, [3000, 5, 700, 0], [3, 1, 8, 0], heads, 2, d, 32, BF, seed=13, tree="tree", stale=float("nan"))
    call("qe_attn_tree_set_split", 0)
    try:
        compare(c, q, seqs, cu, words, *attend(c, q, seqs, cu, 8, mask, lse=True))
    finally:
        call("qe_attn_tree_set_split", 1)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("rows", [5, 16, 17, 32, 33, 128, 129, 256, 257])
def test_row_counts(dev, rows, d, dtype):
    """the rows of a kv head around the sizes at which the kernel changes, over ragged contexts"""
    n = min(rows, 16)
    heads = -(-rows // n)
    c, q, seqs, cu, mask, words = setup(dev, [200, 0, 1000, 65], [n, 1, n - 1, n], heads, 1, d, 16, dtype, seed=rows, tree="random",
                                        stale=float("nan"))
    compare(c, q, seqs, cu, words, *attend(c, q, seqs, cu, n, mask, lse=True))


def test_same_bits_streams_and_graphs(dev):
    """eager calls on two streams, two graphs replayed beside each other, replays with other lengths and masks"""
    c, q, seqs, cu, mask, _ = setup(dev, [3000, 17, 800], [6, 1, 9], 8, 2, 128, 16, BF, seed=14, tree="tree")
    want = attend(c, q, seqs, cu, 9, mask)
    assert torch.equal(want, attend(c, q, seqs, cu, 9, mask))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = attend(c, q, seqs, cu, 9, mask)
    side.synchronize()
    assert torch.equal(want, other)
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    for o in outs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            attend(c, q, seqs, cu, 9, mask, out=o)
            attend(c, q, seqs, cu, 9, mask, out=o)
        graphs.append(graph)
    lib().qe_workspace_count.restype = __import__("ctypes").c_int
    assert call("qe_workspace_count", 5) >= 3  # a stream's and each graph's
    for length in ([3000, 17, 800], [0, 2900, 31], [1, 1, 2999]):
        # every slot's table reaches as far as the first one's: shared pages do for reading
        first = c.table[seqs[0]].clone()
        c.table[:] = first
        full = c.length.clone()
        for s, n in zip(seqs.tolist(), length):
            full[s] = n
        c.length.copy_(full)
        mask.copy_(mask.roll(1))
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        with torch.cuda.stream(a):
            graphs[0].replay()
        with torch.cuda.stream(b):
            graphs[1].replay()
        eager = attend(c, q, seqs, cu, 9, mask)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager) and torch.equal(outs[1], eager), length


def test_nothing_to_do(dev):
    c, q, seqs, cu, _, _ = setup(dev, [5], [1], 2, 1, 64, 16, BF, seed=1)
    assert c.attend(0, q[:0], seqs, ints([0, 0], dev), 1).shape == (0, 2, 64)
    out = torch.full_like(q, 7.0)
    c.attend(0, q, seqs[:0], ints([0], dev), 1, out=out)
    c.attend(0, q, seqs, ints([0, 0], dev), 1, out=out)
    assert (out == 7).all()
