"""The paged cache's operations against the same steps one after the other in Python (attention_ref.Pages): whole numbers
and moved rows have to be equal bit by bit. Then a batch's life through all of them with attention at every step."""
import random

import pytest
import torch

import attention_ref as ref
from qengine_amd import ops

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def make(dev, layers=2, pages=40, page=16, kv=2, d=64, slots=8, tokens=200, dtype=BF, seed=0):
    c = ops.KVCache.empty(layers, pages, page, kv, d, slots, tokens, dtype=dtype, device=dev)
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c.k.copy_(torch.randn(c.k.shape, device=dev, generator=g))
    c.v.copy_(torch.randn(c.v.shape, device=dev, generator=g))
    return c, ref.Pages(c), g


def fill(c, p, lens, dev):
    """slots 0.. with committed tokens"""
    s = list(range(len(lens)))
    assert c.reserve(ints(s, dev), ints(lens, dev)).tolist() == p.reserve(s, lens) == [1] * len(s)
    c.accept(ints(s, dev), ints(lens, dev))
    p.accept(s, lens)
    p.same(values=False)


def test_reserve(dev):
    c, p, _ = make(dev)
    for seqs, add in [([3], [1]), ([0, 5], [16, 33]), ([3, 0], [15, 1]), ([3], [1]), ([1, 2], [0, 0]), ([7, 7, 6], [5, 5, 5]),
                      ([-1, 8, 4], [4, 4, 4]), ([4], [-2]), ([2], [1000]), ([2], [208]), ([6, 1, 0, 2], [208, 208, 500, 1])]:
        assert c.reserve(ints(seqs, dev), ints(add, dev)).tolist() == p.reserve(seqs, add), (seqs, add)
        p.same()


def test_reserve_until_the_pages_run_out(dev):
    """entries are served in order up to the first that does not fit; those that need nothing are done"""
    c, p, _ = make(dev, pages=10, slots=6, tokens=160)
    for seqs, add in [([0, 1, 2], [60, 40, 60]), ([0, 3, 1, 4], [1, 50, 1, 16]), ([4, 5], [16, 16]), ([5, 4], [1, 1]), ([5], [1])]:
        assert c.reserve(ints(seqs, dev), ints(add, dev)).tolist() == p.reserve(seqs, add), (seqs, add)
        p.same()


@pytest.mark.parametrize("pages", [1, 3, 4, 1023, 4096, 70001])
def test_reserve_finds_free_pages_anywhere(dev, pages):
    c = ops.KVCache.empty(1, pages, 16, 1, 64, 4, 16 * 64, device=dev)
    rng = random.Random(pages)
    free = sorted(rng.sample(range(pages), min(pages, 90)))
    c.ref.fill_(1)
    c.ref[torch.tensor(free, device=dev)] = 0
    got = c.reserve(ints([2, 0, 3], dev), ints([16 * 40, 16 * 40, 16 * 10], dev)).tolist()
    want, left = [], len(free)
    total = 0
    for n in (40, 40, 10):
        total += n
        want.append(int(total <= left))
    assert got == want
    taken = [x for s, n, ok in zip((2, 0, 3), (40, 40, 10), want) if ok for x in c.table[s, :n].tolist()]
    assert taken == free[:len(taken)] and c.ref.sum().item() == pages - len(free) + len(taken)


def test_reserve_of_more_than_an_int(dev):
    """1024 entries whose wishes sum past 2^31 pages: those that fit are served, the others refused"""
    c = ops.KVCache.empty(1, 50, 16, 1, 64, 1100, 16, device=dev)
    c = ops.KVCache(c.k, c.v, torch.full((1100, 1 << 22), -1, dtype=torch.int32, device=dev), c.length, c.held, c.ref)
    add = [16 * 10, 16 * 40] + [16 << 22] * 1022
    got = c.reserve(ints(range(1024), dev), ints(add, dev)).tolist()
    assert got == [1, 1] + [0] * 1022 and c.ref.sum().item() == 50 and c.held[:3].tolist() == [10, 40, 0]


@pytest.mark.parametrize("pages,each,first", [(20000, 9, 0), (150000, 20, 0), (5003, 4, 1)])
def test_reserve_of_many_pages(dev, pages, each, first):
    """thousands of pages in one call, scattered over the pool, for 1024 entries of which some name a slot again; the counts
    also where they do not start at 16 bytes"""
    c = ops.KVCache.empty(1, pages, 16, 1, 64, 1200, 16 * 40, device=dev)
    counts = torch.ones(pages + first, dtype=torch.int32, device=dev)[first:]
    c = ops.KVCache(c.k, c.v, c.table, c.length, c.held, counts)
    rng = random.Random(pages)
    free = sorted(rng.sample(range(pages), min(pages * 4 // 5, 1010 * each + 7)))
    counts[torch.tensor(free, device=dev)] = 0
    seqs = rng.sample(range(1200), 1024)
    for i in (1, 2, 3, 4, 5, 64, 127, 500, 1023):  # repeated from one to many places before
        seqs[i] = seqs[rng.randrange(i)]
    got = c.reserve(ints(seqs, dev), ints([16 * each] * 1024, dev)).tolist()
    want, used, table = [], 0, {}
    for i, s in enumerate(seqs):
        ok = s not in seqs[:i]
        if ok:
            used += each
            ok = used <= len(free)
            if ok:
                table[s] = free[used - each:used]
        want.append(int(ok))
    assert got == want
    held, rows = c.held.tolist(), c.table.tolist()
    assert all(rows[s] == table.get(s, []) + [-1] * (40 - len(table.get(s, []))) and held[s] == len(table.get(s, [])) for s in range(1200))
    taken = sum(len(x) for x in table.values())
    assert counts.sum().item() == pages - len(free) + taken and counts.max().item() == 1


def test_reserve_of_many(dev):
    """1024 entries: pages for each, copies for half of them"""
    c, p, _ = make(dev, layers=1, pages=3000, kv=1, slots=1200, tokens=64)
    lens = [17 + i % 20 for i in range(500)]
    fill(c, p, lens, dev)
    kids = list(range(500, 1000))
    assert c.fork(ints(range(500), dev), ints(kids, dev)).tolist() == p.fork(list(range(500)), kids)
    seqs = kids + list(range(1000, 1200)) + list(range(0, 324))
    add = [1 + i % 7 for i in range(1024)]
    assert c.reserve(ints(seqs, dev), ints(add, dev)).tolist() == p.reserve(seqs, add)
    p.same()


def test_fork_shares_and_reserve_copies(dev):
    c, p, _ = make(dev)
    fill(c, p, [37, 32, 0, 5], dev)
    # slots 4.. are children of 0, 1, 0 and of the empty 2; then what is refused
    for par, kid in [([0, 1, 0, 2], [4, 5, 6, 7]), ([0], [4]), ([9, -1, 0], [4, 4, 9]), ([3, 3], [2, 2]), ([3, 2], [2, 7])]:
        assert c.fork(ints(par, dev), ints(kid, dev)).tolist() == p.fork(par, kid), (par, kid)
        p.same()
    # a slot whose page is shared gets a copy, all sharers in one call included; one on its own page does not
    for seqs, add in [([4], [1]), ([0, 6, 5, 1], [1, 2, 3, 1]), ([0], [1]), ([3], [0]), ([7], [20])]:
        assert c.reserve(ints(seqs, dev), ints(add, dev)).tolist() == p.reserve(seqs, add), (seqs, add)
        p.same()


def test_release(dev):
    c, p, _ = make(dev)
    fill(c, p, [37, 32, 20, 5], dev)
    kid = [4, 5]
    c.fork(ints([0, 2], dev), ints(kid, dev)), p.fork([0, 2], kid)
    for seqs, lens in [([0], [33]), ([0], [16]), ([1, 4], [100, 0]), ([2, 2, -1, 99], [3, 0, 0, 0]), ([5], [-4]), ([3, 0], None),
                       ([0, 1, 2, 3, 4, 5, 6, 7], None)]:
        c.release(ints(seqs, dev), None if lens is None else ints(lens, dev))
        p.release(seqs, lens)
        p.same()
    assert not c.ref.any() and not c.held.any()


def test_a_cut_slot_does_not_write_its_siblings_page(dev):
    """a child cut back into a page that its parent holds too gets a copy of it before it may append"""
    c, p, g = make(dev)
    fill(c, p, [32], dev)
    c.fork(ints([0], dev), ints([1], dev)), p.fork([0], [1])
    c.release(ints([1], dev), ints([20], dev)), p.release([1], [20])
    assert c.reserve(ints([1], dev), ints([3], dev)).tolist() == p.reserve([1], [3]) == [1]
    k, v = (torch.randn(3, 2, 64, device=dev, generator=g).to(BF) for _ in range(2))
    c.append(1, k, v, ints([1], dev), ints([0, 3], dev)), p.append(1, k, v, [1], [0, 3])
    p.same()
    assert p.table[0][1] != p.table[1][1] and p.table[0][0] == p.table[1][0]


def test_without_reserve_a_shared_page_stays(dev):
    """rows appended or moved after a fork without a reserve are not written into the page that the parent holds too"""
    c, p, g = make(dev)
    fill(c, p, [20], dev)
    c.fork(ints([0], dev), ints([1], dev)), p.fork([0], [1])
    k, v = (torch.randn(3, 2, 64, device=dev, generator=g).to(BF) for _ in range(2))
    c.append(0, k, v, ints([1], dev), ints([0, 3], dev))
    c.append(None, torch.stack([k, v]), torch.stack([v, k]), ints([0], dev), ints([0, 3], dev))
    c.accept(ints([1], dev), ints([3], dev), ints([[2, 0, 1]], dev)), p.accept([1], [3])
    p.same()


def test_a_path_of_no_columns(dev):
    """commits nothing; the lengths are written all the same"""
    c, p, _ = make(dev)
    fill(c, p, [20, 7], dev)
    after = torch.full_like(c.length, -5)
    c.accept(ints([1, 0], dev), ints([4, 0], dev), torch.empty(2, 0, dtype=torch.int32, device=dev), length=after)
    assert after.tolist() == [20, 7] + [-5] * 6
    c.accept(ints([1, 0], dev), ints([4, 0], dev), torch.empty(2, 0, dtype=torch.int32, device=dev))
    p.same()


@pytest.mark.parametrize("d,kv,page", [(64, 1, 16), (64, 3, 32), (128, 8, 16), (256, 2, 64), (128, 5, 1024)])
def test_append(dev, d, kv, page):
    c, p, g = make(dev, layers=3, pages=24, page=page, kv=kv, d=d, tokens=6 * page, dtype=F16)
    fill(c, p, [page - 1, 0, 2 * page, 5], dev)
    seqs, new = [2, 0, 3, 1, 6], [3, page + 2, 0, 40, 4]
    c.reserve(ints(seqs[:4], dev), ints(new[:4], dev)), p.reserve(seqs[:4], new[:4])  # slot 6 has no page: not written
    cu = [2 + sum(new[:i]) for i in range(6)]
    t = cu[-1] + 5  # rows before and behind the batch
    x = torch.randn(3, t, 2 * kv * d + 8, device=dev, generator=g).to(F16)  # k and v as views of a wider product
    k, v = x[:, :, :kv * d].unflatten(2, (kv, d)), x[:, :, kv * d:2 * kv * d].unflatten(2, (kv, d))
    c.append(1, k[0], v[0], ints(seqs, dev), ints(cu, dev)), p.append(1, k[0], v[0], seqs, cu)
    p.same()
    c.append(None, k, v, ints(seqs, dev), ints(cu, dev)), p.append(None, k, v, seqs, cu)
    p.same()


def test_append_what_is_out_of_range(dev):
    """slots, pages and starts out of range: such rows are not written"""
    c, p, g = make(dev)
    fill(c, p, [10, 20], dev)
    k, v = (torch.randn(6, 2, 64, device=dev, generator=g).to(BF) for _ in range(2))
    c.table[1, 1] = 1 << 30
    p.table[1][1] = 1 << 30
    c.append(0, k, v, ints([-1, 8, 0, 1], dev), ints([0, 1, 2, 3, 6], dev))
    p.append(0, k[2:3], v[2:3], [0], [0, 1])
    p.same()


def test_append_to_many(dev):
    n = 300
    c, p, g = make(dev, layers=1, pages=700, kv=1, slots=n, tokens=32)
    fill(c, p, [i % 17 for i in range(n)], dev)
    new = [i % 3 for i in range(n)]
    c.reserve(ints(range(n), dev), ints(new, dev)), p.reserve(list(range(n)), new)
    cu = [sum(new[:i]) for i in range(n + 1)]
    k, v = (torch.randn(cu[-1], 1, 64, device=dev, generator=g).to(BF) for _ in range(2))
    c.append(0, k, v, ints(range(n), dev), ints(cu, dev)), p.append(0, k, v, list(range(n)), cu)
    p.same()


@pytest.mark.parametrize("d,kv,page", [(64, 1, 16), (128, 5, 16), (256, 2, 32), (64, 8, 128)])
def test_accept(dev, d, kv, page):
    """paths of any order, with repeats, with rows that stay, with entries out of range, up to 64 long"""
    c, p, _ = make(dev, layers=3, pages=60, page=page, kv=kv, d=d, tokens=200)
    lens = [0, 15, 16, 30, 7, 100]
    fill(c, p, lens, dev)
    seqs = [3, 0, 5, 1, 2, 4]
    c.reserve(ints(seqs, dev), ints([64] * 6, dev)), p.reserve(seqs, [64] * 6)
    paths = [[0, 2, 5, 9], [3, 1, 2, 0], [1, 1, 1, 63], [0, 1, 2, 3], [-1, 64, 5, 4000], [7, 6, 5, 4]]
    count = [4, 4, 3, 2, 4, 9]
    before = c.length.clone()
    after = before.clone()
    p_after = list(p.length)
    p.accept(seqs, count, paths, length=p_after)
    c.accept(ints(seqs, dev), ints(count, dev), ints(paths, dev), length=after)
    assert torch.equal(c.length, before) and after.tolist() == p_after
    p.same()
    order = random.Random(1).sample(range(64), 64)
    c.accept(ints([3], dev), ints([64], dev), ints([order], dev)), p.accept([3], [64], [order])
    p.same()
    c.accept(ints([0, 77, 5], dev), ints([-3, 1, 10 ** 6], dev)), p.accept([0, 77, 5], [-3, 1, 10 ** 6])
    p.same()


def test_a_step_in_a_graph(dev):
    """release, fork, reserve, append and accept captured once and replayed against the same steps in Python"""
    c, p, g = make(dev, pages=64)
    fill(c, p, [21, 40], dev)
    par, kid, one = ints([0, 1, 0], dev), ints([2, 3, 4], dev), ints([1, 1, 1], dev)
    k, v = (torch.randn(2, 3, 2, 64, device=dev, generator=g).to(BF) for _ in range(2))
    cu = ints([0, 1, 2, 3], dev)

    def step():
        c.release(kid)
        a = c.fork(par, kid)
        b = c.reserve(kid, one)
        c.append(None, k, v, kid, cu)
        c.accept(kid, one)
        return a, b

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ok = step()
    for order in ([0, 1, 0], [1, 1, 1], [0, 0, 7]):
        par.copy_(ints(order, dev))
        k.normal_(generator=g), v.normal_(generator=g)
        graph.replay()
        torch.cuda.synchronize()
        kids = [2, 3, 4]
        p.release(kids)
        assert ok[0].tolist() == p.fork(order, kids) and ok[1].tolist() == p.reserve(kids, [1] * 3)
        p.append(None, k, v, kids, [0, 1, 2, 3])
        p.accept(kids, [1] * 3)
        p.same()


def attention(state, layer, s, q, first, group):
    """64-bit rows of one slot's tokens first.. (a chain) over all before, per head"""
    x, heads, d = q.shape
    k, v = state.tokens(layer, s, first + x)
    seen = torch.ones(x, first + x, dtype=torch.bool, device=q.device).tril(first)
    return [ref.rows(q[:, h], k[:, h // group], v[:, h // group], seen, d ** -0.5) for h in range(heads)]


def test_a_batch_from_prompt_to_drafts(dev):
    """two prompts through attn_prompt, a decoded token, a fork, a drafted tree verified and its path accepted, a decoded
    token after it, a release: every attention against 64 bits over what the slots then hold"""
    kv, group, d, layers = 2, 3, 128, 2
    c, p, g = make(dev, layers=layers, pages=60, page=16, kv=kv, d=d, slots=6, tokens=160)

    def rows(n):
        return (torch.randn(n, kv * group, d, device=dev, generator=g).to(BF), torch.randn(n, kv, d, device=dev, generator=g).to(BF),
                torch.randn(n, kv, d, device=dev, generator=g).to(BF))

    def grow(seqs, new):
        cu = [sum(new[:i]) for i in range(len(new) + 1)]
        assert c.reserve(ints(seqs, dev), ints(new, dev)).tolist() == p.reserve(seqs, new) == [1] * len(seqs)
        return cu

    def put(layer, k, v, seqs, cu):
        c.append(layer, k, v, ints(seqs, dev), ints(cu, dev)), p.append(layer, k, v, seqs, cu)

    def commit(seqs, n, path=None):
        c.accept(ints(seqs, dev), ints(n, dev), None if path is None else ints(path, dev)), p.accept(seqs, n, path)
        p.same()

    def decode(seqs):
        cu = grow(seqs, [1] * len(seqs))
        for layer in range(layers):
            q, k, v = rows(len(seqs))
            put(layer, k, v, seqs, cu)
            o = c.attend(layer, q, ints(seqs, dev), ints(cu, dev), 1)
            for b, s in enumerate(seqs):
                for h, w in enumerate(attention(p, layer, s, q[b:b + 1], p.length[s], group)):
                    ref.check(o[b:b + 1, h], None, *w, what=f"decode {s} {layer} {h}")
        commit(seqs, [1] * len(seqs))

    seqs, lens = [4, 1], [75, 18]
    cu = grow(seqs, lens)
    for layer in range(layers):
        q, k, v = rows(sum(lens))
        put(layer, k, v, seqs, cu)
        o = ops.attn_prompt(q, k, v, ints(cu, dev))
        for b, s in enumerate(seqs):
            for h, w in enumerate(attention(p, layer, s, q[cu[b]:cu[b + 1]], 0, group)):
                ref.check(o[cu[b]:cu[b + 1], h], None, *w, what=f"prompt {s} {layer} {h}")
    commit(seqs, lens)
    decode([1, 4])
    assert c.fork(ints([4, 4], dev), ints([0, 5], dev)).tolist() == p.fork([4, 4], [0, 5]) == [1, 1]
    decode([5, 1, 0])  # the children copy the shared page, the parent's stays
    # a tree of 7 on slot 0 (node 0 the root, 1 2 3 its children, 4 5 under 2, 6 under 5), a chain of 3 on slot 4
    parent = [-1, 0, 0, 0, 2, 2, 5]
    words = []
    for i, up in enumerate(parent):
        words.append((words[up] if up >= 0 else 0) | 1 << i)
    words += [1, 3, 7]
    seqs, new = [0, 4], [7, 3]
    cu = grow(seqs, new)
    qs = []
    for layer in range(layers):
        q, k, v = rows(10)
        put(layer, k, v, seqs, cu)
        o = c.attend(layer, q, ints(seqs, dev), ints(cu, dev), 7, mask=torch.tensor(words, device=dev))
        for b, s in enumerate(seqs):
            n, x = p.length[s], new[b]
            k, v = p.tokens(layer, s, n + x)
            seen = torch.ones(x, n + x, dtype=torch.bool)
            for i in range(x):
                seen[i, n:] = torch.tensor([bool(words[cu[b] + i] >> j & 1) for j in range(x)])
            for h in range(kv * group):
                w = ref.rows(q[cu[b]:cu[b + 1], h], k[:, h // group], v[:, h // group], seen.to(dev), d ** -0.5)
                ref.check(o[cu[b]:cu[b + 1], h], None, *w, what=f"tree {s} {layer} {h}")
        qs.append((q, o))
    commit(seqs, [4, 2], [[0, 2, 5, 6], [0, 1, 2, 0]])
    # the accepted path is a chain now: its last row's attention is what the tree gave it
    for layer, (q, o) in enumerate(qs):
        for h, w in enumerate(attention(p, layer, 0, q[6:7], p.length[0] - 1, group)):
            ref.check(o[6:7, h], None, *w, what=f"path {layer} {h}")
    decode([0, 4, 5, 1])
    c.release(ints([0, 5, 4, 1], dev)), p.release([0, 5, 4, 1])
    p.same()
    assert not c.ref.any()
