"""Attention over prompts and over a paged cache, and the cache's own operations, measured as a serving program calls them.

With `own` false `run` computes them in elementary torch operations in 32 bits, rounded once at the end; with `own` true it
calls the framework (`qengine_amd.ops`). A case is a dict of plain values; lengths of ragged batches follow from the case
alone, values, page tables and trees from the seed.

Kinds:
  prompt  causal attention over packed prompts with grouped heads (ops.attn_prompt)
  tree    attention of drafted tokens, one (decode) or a tree of them, over a paged cache (KVCache.attend)
  append  new keys and values into the cache's pages, one layer or all (KVCache.append)
  beam    one step of sampling in parallel: the last step's children are released, the parents forked into them, room for the
          next token reserved, which copies the partly filled pages (KVCache.release, fork, reserve)
  accept  the cache's side of a verified draft, all layers: drafted rows appended, the accepted path moved together
          (KVCache.append, accept)

A cache holds k, v [layers, pages, kv heads, page, d], table [sequences, pages of one] (-1: none), length (tokens), held
(pages) [sequences] and ref [pages] (sequences that hold a page, 0: free).
"""
import math
import random

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    # 40 heads of 128 over 8 are a hidden size of 5120, 16 of 128 a hidden size of 2048 (bench.py's matrices)
    big = {"heads": 40, "kv": 8, "d": 128, "dtype": "bf16"}
    return [
        # the first chat turn of one user
        {"name": "prompt_1x300", "kind": "prompt", "seqs": 1, "tokens": 300, "tail": 0, **big},
        # a server's prefill batch: prompts of many lengths packed without padding, a few rows left over at the end
        {"name": "prompt_20_packed", "kind": "prompt", "seqs": 20, "tokens": 8191, "tail": 9, **big},
        # one long document, wide heads
        {"name": "prompt_1x16384", "kind": "prompt", "seqs": 1, "tokens": 16384, "tail": 0, "heads": 16, "kv": 2, "d": 256,
         "dtype": "f16"},
        # one sequence generating: the latency of a token
        {"name": "decode_1", "kind": "tree", "seqs": 1, "context": 2100, "nodes": 1, "page": 16, **big},
        # a busy server's decode batch, contexts of all lengths
        {"name": "decode_64", "kind": "tree", "seqs": 64, "context": 8000, "nodes": 1, "page": 64, **big},
        # drafted trees of a dozen sequences verified together
        {"name": "verify_12x32", "kind": "tree", "seqs": 12, "context": 6000, "nodes": 32, "page": 32, **big},
        # two sequences deep in long documents with short drafts
        {"name": "verify_long_2x5", "kind": "tree", "seqs": 2, "context": 131072, "nodes": 5, "page": 128, "heads": 16, "kv": 2,
         "d": 256, "dtype": "f16"},
        # one layer's new rows of a decode batch
        {"name": "append_64x1", "kind": "append", "seqs": 64, "tokens": 64, "layers": 1, "page": 64, **big},
        # all layers of a prompt that another machine prefilled
        {"name": "append_2048_all", "kind": "append", "seqs": 3, "tokens": 2048, "layers": 32, "page": 32, **big},
        # four beams of one sequence
        {"name": "beam_4", "kind": "beam", "seqs": 1, "children": 4, "context": 1000, "layers": 32, "page": 16, **big},
        # eight samples each of a dozen prompts
        {"name": "beam_12x8", "kind": "beam", "seqs": 12, "children": 8, "context": 3000, "layers": 16, "page": 64, **big},
        # the drafts of a batch after their verification
        {"name": "accept_16x24", "kind": "accept", "seqs": 16, "nodes": 24, "context": 2000, "layers": 32, "page": 32, **big},
    ]


MOST_BYTES = 1.1e9
MOST_FLOPS = 2.3e12


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "prompt", "tree", "tree", "tree", "tree", "append", "beam", "accept"])
    while True:
        kv = rng.choice([1, 2, 4, 8])
        c = {"kind": kind, "heads": kv * rng.choice([1, 2, 4, 5, 7, 8]), "kv": kv, "d": rng.choice([64, 128, 128, 256]),
             "dtype": rng.choice(["bf16", "bf16", "f16"])}
        if kind == "prompt":
            c["seqs"] = _log(rng, 1, 48)
            c["tokens"] = c["seqs"] * _log(rng, 1, 4096) + rng.randint(0, 63)
            c["tail"] = rng.choice([0, 0, rng.randint(1, 40)])
            if c["tokens"] > 16384:
                continue
        else:
            c["page"] = rng.choice([16, 32, 64, 128])
            c["seqs"] = _log(rng, 1, 96)
        if kind == "tree":
            c.update(context=_log(rng, 1, 65536), nodes=rng.choice([1, 1, 1, 2, 4, rng.randint(3, 64)]))
        elif kind == "append":
            c.update(tokens=c["seqs"] + _log(rng, 1, 4096), layers=rng.choice([1, 1, 8, 24]))
        elif kind == "beam":
            c.update(children=rng.randint(1, 8), context=_log(rng, 1, 4096), layers=rng.choice([4, 12, 24]))
            c["seqs"] = min(c["seqs"], 12)
        elif kind == "accept":
            c.update(nodes=rng.randint(2, 64), context=_log(rng, 1, 2048), layers=rng.choice([4, 12, 24]))
            c["seqs"] = min(c["seqs"], 24)
        w = work(c)
        plain = 0  # what the plain forms hold of scores or of the cache, in values
        if kind == "prompt":
            plain = c["seqs"] * c["heads"] * max(_prompt_lens(c)) ** 2
        elif kind == "tree":
            plain = c["seqs"] * c["context"] * (c["kv"] * c["d"] + c["heads"] * c["nodes"])
        pool = 2 * c.get("layers", 1) * _pages(c) * c["page"] * c["kv"] * c["d"] if kind != "prompt" else 0
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS and plain < 4.5e9 and pool < 2.2e9:
            return c


def _own_rng(case):
    return random.Random("/".join("%s=%s" % (k, case[k]) for k in sorted(case) if k != "name"))


def _prompt_lens(case):
    """lengths that sum to the packed tokens: most short, a few long, some empty where the batch is padded"""
    rng = _own_rng(case)
    n, total = case["seqs"], case["tokens"]
    if n == 1:
        return [total]
    w = [math.exp(rng.gauss(0, 0.9)) for _ in range(n)]
    lens = [int(total * x / sum(w)) for x in w]
    lens[rng.randrange(n)] += total - sum(lens)
    return lens


def _contexts(case):
    """committed tokens of each sequence: up to `context`, one of them that long"""
    rng = _own_rng(case)
    n, most = case["seqs"], case["context"]
    c = [max(0, int(most * (1 - 0.9 * rng.random() ** 1.5))) for _ in range(n)]
    c[rng.randrange(n)] = most
    return c


def _new_tokens(case):
    """rows that each sequence brings: drafted nodes, or its part of the appended tokens"""
    rng = _own_rng(case)
    rng.random()
    if case["kind"] in ("tree", "accept"):
        k = case["nodes"]
        return [k if rng.random() < 0.5 else rng.randint((k + 1) // 2, k) for _ in range(case["seqs"])]
    n, total = case["seqs"], case["tokens"]
    cuts = sorted(rng.randint(0, total - n) for _ in range(n - 1))
    return [b - a + 1 for a, b in zip([0] + cuts, cuts + [total - n])]


def _lens(case):
    """(committed tokens, new tokens) of each sequence of a cache"""
    if case["kind"] == "append":
        new = _new_tokens(case)
        rng = _own_rng(case)
        return [rng.randint(0, 900) for _ in new], new
    if case["kind"] == "beam":
        return _contexts(case), [0] * case["seqs"]
    return _contexts(case), _new_tokens(case)


def _accepted(case):
    rng = _own_rng(case)
    return [rng.randint(1, min(k, 8)) for k in _new_tokens(case)]


def _pages(case):
    """pages of the pool: what the sequences hold, room to fork, and a quarter free"""
    ctx, new = _lens(case)
    p = case["page"]
    used = sum(-(-(c + n) // p) for c, n in zip(ctx, new))
    if case["kind"] == "beam":
        used += 2 * case["seqs"] * case["children"]
    return used + used // 4 + 8


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    rng = random.Random(int(seed))
    dt = DT[case["dtype"]]
    h, kv, d = case["heads"], case["kv"], case["d"]

    def rows(*shape):
        return torch.randn(*shape, device=DEV, generator=g, dtype=torch.float32).to(dt)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def starts(lens):
        return ints([sum(lens[:i]) for i in range(len(lens) + 1)])

    if case["kind"] == "prompt":
        lens, t = _prompt_lens(case), case["tokens"] + case["tail"]
        qkv = rows(t, (h + 2 * kv) * d)  # one fused product's rows; q, k and v are views of it
        q, k, v = (x.view(t, -1, d) for x in qkv.split([h * d, kv * d, kv * d], dim=1))
        return {"case": case, "q": q, "k": k, "v": v, "cu": starts(lens), "out": torch.zeros(t, h, d, dtype=dt, device=DEV)}

    ctx, new = _lens(case)
    page, pages, layers = case["page"], _pages(case), case.get("layers", 1)
    kids = case.get("children", 0)
    n = len(ctx)
    slots = n + n * kids
    width = -(-(max(c + x for c, x in zip(ctx, new)) + 1) // page) + 1
    order = list(range(pages))
    rng.shuffle(order)  # a pool that has been in use: no two pages of a sequence follow each other
    place = list(range(slots))
    rng.shuffle(place)
    table = [[-1] * width for _ in range(slots)]
    length, held, ref, at = [0] * slots, [0] * slots, [0] * pages, 0
    for i, (c, x) in enumerate(zip(ctx, new)):
        s, k = place[i], -(-(c + x) // page)
        table[s][:k] = order[at:at + k]
        for p in order[at:at + k]:
            ref[p] = 1
        length[s], held[s], at = c, k, at + k
    s = {"case": case, "k": rows(layers, pages, kv, page, d), "v": rows(layers, pages, kv, page, d), "table": ints(table),
         "length": ints(length), "held": ints(held), "ref": ints(ref), "seqs": ints(place[:n])}
    if case["kind"] == "beam":
        s["parents"] = ints([place[rng.randrange(n)] if rng.random() < 0.5 else place[i // kids] for i in range(n * kids)])
        s["children"] = ints(place[n:])
        s["one"] = ints([1] * (n * kids))
        return s
    s["cu"] = starts(new)
    if case["kind"] == "tree":
        s["q"] = rows(sum(new), h, d)
        s["mask"], masks = None, []
        if case["nodes"] > 1:
            for x in new:  # node i hangs on the root or on an earlier node; a node sees itself and its ancestors
                seen = []
                for i in range(x):
                    above = rng.randint(max(-1, i - 6), i - 1) if i else -1
                    seen.append((seen[above] if above >= 0 else 0) | 1 << i)
                masks += [m - (1 << 64) if m >> 63 else m for m in seen]
            s["mask"] = torch.tensor(masks, dtype=torch.int64, device=DEV)
        return s
    s["new_k"], s["new_v"] = rows(layers, sum(new), kv, d), rows(layers, sum(new), kv, d)
    if case["kind"] == "accept":
        count = _accepted(case)
        most = max(count)
        path = [sorted(rng.sample(range(x), a)) + [0] * (most - a) for x, a in zip(new, count)]
        s["path"], s["count"], s["after"] = ints(path), ints(count), s["length"].clone()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _run_own(s) if own else _PLAIN[s["case"]["kind"]](s)


def _run_own(s):
    from qengine_amd import ops
    kind = s["case"]["kind"]
    if kind == "prompt":
        return ops.attn_prompt(s["q"], s["k"], s["v"], s["cu"], out=s["out"])
    if "cache" not in s:  # the handle that a server keeps for as long as the pool lives
        s["cache"] = ops.KVCache(s["k"], s["v"], s["table"], s["length"], s["held"], s["ref"])
    cache = s["cache"]
    if kind == "tree":
        return cache.attend(0, s["q"], s["seqs"], s["cu"], s["case"]["nodes"], mask=s["mask"])
    if kind == "append":
        cache.append(None, s["new_k"], s["new_v"], s["seqs"], s["cu"])
        return {"k": s["k"], "v": s["v"]}
    if kind == "accept":
        cache.append(None, s["new_k"], s["new_v"], s["seqs"], s["cu"])
        cache.accept(s["seqs"], s["count"], s["path"], length=s["after"])
        return {"k": s["k"], "v": s["v"], "length": s["after"]}
    cache.release(s["children"])
    forked = cache.fork(s["parents"], s["children"])
    got = cache.reserve(s["children"], s["one"])
    return {"k": s["k"], "v": s["v"], "table": s["table"], "length": s["length"], "held": s["held"], "ref": s["ref"],
            "forked": forked, "got": got}


# ---- the plain forms
def _softmax_times(scores, seen, v):
    """softmax over the seen places times v; rows that see nothing give zeros"""
    scores = scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    return (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _plain_prompt(s):
    c, cu = s["case"], s["cu"].long()
    h, kv, d = c["heads"], c["kv"], c["d"]
    t, n, most = s["q"].shape[0], c["seqs"], max(_prompt_lens(c))
    at = torch.arange(most, device=DEV)
    idx = cu[:-1, None] + at                         # [n, most] rows of a padded batch
    live = at < (cu[1:] - cu[:-1])[:, None]
    idx = torch.where(live, idx, torch.zeros_like(idx))
    q = s["q"].float()[idx].view(n, most, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, d)
    k = s["k"].float()[idx].permute(0, 2, 3, 1).contiguous()
    v = s["v"].float()[idx].permute(0, 2, 1, 3).contiguous()
    scores = (q @ k).mul_(d ** -0.5).view(n, kv, h // kv, most, most)
    seen = (at[None, :] <= at[:, None])[None] & live[:, None, :]
    o = _softmax_times(scores, seen[:, None, None], v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, h, d).to(s["q"].dtype)
    out = torch.zeros(t + 1, h, d, dtype=o.dtype, device=DEV)
    out[torch.where(live, idx, torch.full_like(idx, t))] = o  # rows past a sequence's end go to a row that is dropped
    return out[:t]


def _plain_tree(s):
    c, cu = s["case"], s["cu"].long()
    h, kv, d, page, n, most = c["heads"], c["kv"], c["d"], c["page"], c["seqs"], c["nodes"]
    g = h // kv
    length = s["length"].long()[s["seqs"].long()]
    new = cu[1:] - cu[:-1]
    at = torch.arange(c["context"] + most, device=DEV)
    live = at < (length + new)[:, None]
    ids = s["table"].long()[s["seqs"].long()]
    pg = torch.where(live, ids.gather(1, (at // page).clamp_max(ids.shape[1] - 1).expand(n, -1)), torch.zeros_like(at))
    k = s["k"][0].permute(0, 2, 1, 3)[pg, (at % page).expand(n, -1)].float().permute(0, 2, 3, 1).contiguous()
    v = s["v"][0].permute(0, 2, 1, 3)[pg, (at % page).expand(n, -1)].float().permute(0, 2, 1, 3).contiguous()
    i = torch.arange(most, device=DEV)
    has = i < new[:, None]
    row = torch.where(has, cu[:-1, None] + i, torch.zeros_like(i))
    q = s["q"].float()[row].view(n, most, kv, g, d).permute(0, 2, 3, 1, 4).reshape(n, kv, g * most, d)
    scores = (q @ k).mul_(d ** -0.5).view(n, kv, g, most, -1)
    j = at[None, :] - length[:, None]                # place among the drafted tokens
    bit = j.clamp(0, 63)[:, None, :]
    if s["mask"] is None:
        tree = j[:, None, :] <= i[None, :, None]
    else:
        tree = (s["mask"][row][:, :, None] >> bit & 1) > 0
    seen = ((j < 0)[:, None, :] | tree) & live[:, None, :]
    o = _softmax_times(scores, seen[:, None, None], v[:, :, None])
    o = o.permute(0, 3, 1, 2, 4).reshape(n, most, h, d).to(s["q"].dtype)
    out = torch.zeros(s["q"].shape[0] + 1, h, d, dtype=o.dtype, device=DEV)
    out[torch.where(has, row, torch.full_like(row, s["q"].shape[0]))] = o
    return out[:-1]


def _places(s, pos, slot):
    """(page, row in it) of tokens at `pos` of sequences `slot`"""
    p = s["case"]["page"]
    return s["table"].long()[slot, pos // p], pos % p


def _put_new(s):
    cu, slot = s["cu"].long(), s["seqs"].long()
    t = torch.arange(s["new_k"].shape[1], device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    pg, off = _places(s, s["length"].long()[slot[b]] + t - cu[b], slot[b])
    s["k"].permute(1, 3, 0, 2, 4)[pg, off] = s["new_k"].permute(1, 0, 2, 3)
    s["v"].permute(1, 3, 0, 2, 4)[pg, off] = s["new_v"].permute(1, 0, 2, 3)


def _plain_append(s):
    _put_new(s)
    return {"k": s["k"], "v": s["v"]}


def _move(x, to_pg, to_off, from_pg, from_off):
    x[to_pg, to_off] = x[from_pg, from_off]


def _plain_accept(s):
    _put_new(s)
    slot, count = s["seqs"].long(), s["count"].long()
    j = torch.arange(s["path"].shape[1], device=DEV)
    src = torch.where(j < count[:, None], s["path"].long(), j)
    first = s["length"].long()[slot][:, None]
    from_pg, from_off = _places(s, first + src, slot[:, None])
    # places past a sequence's drafted tokens are written to themselves
    spare = (first + j) // s["case"]["page"] >= s["held"].long()[slot][:, None]
    to_pg, to_off = _places(s, torch.where(spare, first, first + j), slot[:, None])
    from_pg, from_off = torch.where(spare, from_pg[:, :1], from_pg), torch.where(spare, from_off[:, :1], from_off)
    _move(s["k"].permute(1, 3, 0, 2, 4), to_pg, to_off, from_pg, from_off)
    _move(s["v"].permute(1, 3, 0, 2, 4), to_pg, to_off, from_pg, from_off)
    after = s["after"]
    after[slot] = (first[:, 0] + count).int()
    return {"k": s["k"], "v": s["v"], "length": after}


def _merge(x, to, old, part):
    x[to] = torch.where(part, x[old], x[to])


def _plain_beam(s):
    page, width = s["case"]["page"], s["table"].shape[1]
    kids, par = s["children"].long(), s["parents"].long()
    table, length, held, ref = s["table"], s["length"], s["held"], s["ref"]
    col = torch.arange(width, device=DEV)

    def count(rows, has, by):
        ref.index_add_(0, rows.clamp_min(0).flatten().long(), (has.int() * by).flatten().int())

    # release
    count(table[kids], col < held[kids][:, None], -1)
    table[kids], length[kids], held[kids] = -1, 0, 0
    # fork: every page that holds a committed token is shared
    keep = (length[par] + page - 1) // page
    rows = torch.where(col < keep[:, None], table[par], -1)
    table[kids], length[kids], held[kids] = rows, length[par], keep
    count(rows, col < keep[:, None], 1)
    # reserve one token: a new page where the last one is full, a copy of the page where it is shared
    at = length[kids].long() // page
    off = length[kids].long() % page
    old = table[kids, at].long()
    copy = (off > 0) & (ref[old.clamp_min(0)] > 1)
    need = ((length[kids] + page) // page - held[kids]).clamp_min(0).long() + copy
    last = need.cumsum(0)
    free = torch.argsort((ref > 0).int(), stable=True)
    got = (need == 0) | (last <= (ref == 0).sum())
    fresh = free[(last - need).clamp_max(free.shape[0] - 1)]
    new_id = torch.where(got & (need > 0), fresh, old)
    pos = torch.arange(page, device=DEV)
    part = (copy & got)[:, None] & (pos < off[:, None])
    part = part[:, None, None, :, None]
    _merge(s["k"].transpose(0, 1), new_id, old, part)
    _merge(s["v"].transpose(0, 1), new_id, old, part)
    table[kids, at] = new_id.int()
    held[kids] += (need - copy.long()).int() * got
    ref.index_add_(0, new_id, (got & (need > 0)).int())
    ref.index_add_(0, old.clamp_min(0), -(copy & got).int())
    return {"k": s["k"], "v": s["v"], "table": table, "length": length, "held": held, "ref": ref,
            "forked": torch.ones_like(s["children"]), "got": got.int()}


_PLAIN = {"prompt": _plain_prompt, "tree": _plain_tree, "append": _plain_append, "accept": _plain_accept, "beam": _plain_beam}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "prompt":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        cu = s["cu"].tolist()
        for a, b in zip(cu[:-1], cu[1:]):
            for h in range(case["heads"]):
                m = h * case["kv"] // case["heads"]
                for r in range(a, b, 2048):
                    e = min(b, r + 2048)
                    x = s["q"][r:e, h].double() @ s["k"][a:e, m].double().T / math.sqrt(case["d"])
                    x += torch.full_like(x, -math.inf).triu(r - a + 1)
                    out[r:e, h] = torch.softmax(x, 1) @ s["v"][a:e, m].double()
        return out
    table, length = s["table"].tolist(), s["length"].tolist()
    seqs, page = s["seqs"].tolist(), case["page"]
    if kind == "tree":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
        cu = s["cu"].tolist()
        for b, slot in enumerate(seqs):
            c, n = length[slot], cu[b + 1] - cu[b]
            ids = torch.tensor(table[slot][:-(-(c + n) // page)], device=DEV)
            seen = torch.ones(n, c + n, dtype=torch.bool)
            if s["mask"] is None:
                seen[:, c:] = torch.ones(n, n).tril().bool()
            else:
                m = s["mask"][cu[b]:cu[b + 1]].tolist()
                seen[:, c:] = torch.tensor([[x >> j & 1 for j in range(n)] for x in m]).bool()
            for h in range(case["heads"]):
                m = h * case["kv"] // case["heads"]
                k = s["k"][0, ids, m].double().reshape(-1, case["d"])[:c + n]
                v = s["v"][0, ids, m].double().reshape(-1, case["d"])[:c + n]
                x = s["q"][cu[b]:cu[b + 1], h].double() @ k.T / math.sqrt(case["d"])
                out[cu[b]:cu[b + 1], h] = torch.softmax(x.masked_fill(~seen.to(DEV), -math.inf), 1) @ v
        return out
    k, v = s["k"].clone(), s["v"].clone()
    if kind in ("append", "accept"):
        cu = s["cu"].tolist()
        moves = []
        for b, slot in enumerate(seqs):
            new = list(range(cu[b], cu[b + 1]))
            if kind == "accept":
                path = s["path"][b].tolist()[:int(s["count"][b])]
                new[:len(path)] = [cu[b] + i for i in path]  # what each drafted place holds afterwards
            moves += [(table[slot][(length[slot] + i) // page], (length[slot] + i) % page, t) for i, t in enumerate(new)]
        pg, off, t = (torch.tensor(x, device=DEV) for x in zip(*moves))
        for pool, rows in ((k, s["new_k"]), (v, s["new_v"])):
            for layer in range(pool.shape[0]):
                pool[layer].transpose(1, 2)[pg, off] = rows[layer][t]
        if kind == "append":
            return {"k": k, "v": v}
        return {"k": k, "v": v, "length": None}
    held, ref = s["held"].tolist(), s["ref"].tolist()
    kids, par = s["children"].tolist(), s["parents"].tolist()
    for c, p in zip(kids, par):  # the children hold nothing at first
        used = -(-length[p] // page)
        table[c][:used] = table[p][:used]
        length[c], held[c] = length[p], used
        for q in table[p][:used]:
            ref[q] += 1
    was, taken = list(ref), list(ref)
    for c in kids:
        full, off = divmod(length[c], page)
        old = table[c][full]
        if off == 0 or was[old] > 1:
            new = taken.index(0)
            taken[new] = 1
            if off:
                k[:, new, :, :off], v[:, new, :, :off] = k[:, old, :, :off], v[:, old, :, :off]
    return {"k": k, "v": v, "table": None, "length": None, "held": None, "ref": None, "forked": None, "got": None}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    h, kv, d = case["heads"], case["kv"], case["d"]
    if case["kind"] == "prompt":
        lens = _prompt_lens(case)
        return {"bytes": 2.0 * sum(lens) * (2 * h + 2 * kv) * d, "flops": 4.0 * d * h * sum(x * (x + 1) // 2 for x in lens)}
    ctx, new = _lens(case)
    row = 2.0 * 2 * kv * d  # bytes of one token's keys and values in one layer
    if case["kind"] == "tree":
        cells = sum(n * c + n * (n + 1) / 2 for c, n in zip(ctx, new))
        return {"bytes": sum(c + n for c, n in zip(ctx, new)) * row + 2.0 * 2 * sum(new) * h * d, "flops": 4.0 * d * h * cells}
    layers = case["layers"]
    if case["kind"] == "append":
        return {"bytes": 2 * layers * sum(new) * row, "flops": 0.0}
    if case["kind"] == "accept":
        return {"bytes": 2 * layers * (sum(new) + sum(_accepted(case))) * row, "flops": 0.0}
    # the children's tables and references, and the copied rows of the partly filled pages (as if every parent forked alike)
    page, kids = case["page"], case["children"]
    return {"bytes": sum(kids * (2 * layers * (c % page) * row + 16.0 * (c // page + 1)) for c in ctx), "flops": 0.0}
