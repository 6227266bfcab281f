"""Attention and the paged cache in 64 bits and plain Python, for the tests, with the error bound of the kernels.

Bound of an output o = sum_j p_j v_j / sum_j p_j, u = half a step of the values' type (2^-8 bf16, 2^-11 fp16):
  * the probabilities are rounded to the type for the second product: at most u sum p |v| / sum p;
  * a score is an fp32 sum of d exact products: off by at most (d + 2) 2^-24 sum |q k| scale, its exponential by that (relative)
    and by 2^-17 more (the exponent's own rounding, below 2^6 in base 2 here, and v_exp_f32); the fp32 sums over n keys add
    at most n 2^-24; all of them relative to sum p |v| / sum p, twice (numerator and denominator);
  * an fp16 probability below 2^-14 is off by up to 2^-25 and the largest one is at least 1: n 2^-25 max |v|;
  * the result is rounded: u |o|, or half of the smallest subnormal (2^-25 fp16).
"""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def rows(q, k, v, seen, scale):
    """q [r][d], k, v [n][d] (16-bit), seen [r][n] -> (o, lse, bound of o, bound of lse) in 64 bits"""
    u = HALF_STEP[q.dtype]
    n, d = k.shape
    qd, kd, vd = q.double(), k.double(), v.double()
    # what no row of the call may see must not matter: a row's own sums run over its own keys alone
    any_seen = seen.any(0)
    kd = torch.where(any_seen[:, None], kd, torch.zeros_like(kd))
    vd = torch.where(any_seen[:, None], vd, torch.zeros_like(vd))
    s = (qd @ kd.T * scale).masked_fill(~seen, -math.inf)
    top = s.amax(1, keepdim=True) if n else torch.full((len(q), 1), -math.inf, dtype=torch.float64, device=q.device)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    l = p.sum(1, keepdim=True)
    ls = l.clamp_min(1e-300)
    o, a = p @ vd / ls, p @ vd.abs() / ls
    e = ((d + 2) * 2.0 ** -24 * scale * (qd.abs() @ kd.abs().T).amax(1, keepdim=True) if n else torch.zeros_like(l)) + 2.0 ** -17 + n * 2.0 ** -24
    big = vd.abs().max() if n else 0.0
    bound = (u + 2 * e) * 1.02 * a + u * o.abs() * 1.02 + (n * 2.0 ** -25 * big + 2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    lse = torch.where(l > 0, top + torch.log(ls), torch.full_like(l, -math.inf))
    return o, lse[:, 0], bound, (e + 2.0 ** -22 * (1 + lse.abs()))[:, 0]


def check(out, lse, o, l, ob, lb, what=""):
    out = out.double()
    assert torch.isfinite(out).all(), what
    over = (out - o).abs() - ob
    assert over.max() <= 0, f"{what}: off by {((out - o).abs() / ob.clamp_min(1e-30)).max().item():.3f} bounds at {over.argmax().item()}"
    if lse is not None:
        empty = torch.isinf(l)
        assert torch.equal(torch.isinf(lse) & (lse < 0), empty), what
        assert ((lse.double() - l).abs()[~empty] <= lb[~empty]).all(), what


class Pages:
    """the cache's bookkeeping, one step after the other"""

    def __init__(self, cache):
        self.c = cache
        self.table, self.length, self.held, self.ref = (x.tolist() for x in (cache.table, cache.length, cache.held, cache.ref))
        self.k, self.v = cache.k.clone(), cache.v.clone()
        self.page, self.width, self.slots = cache.page, cache.width, cache.slots

    def reserve(self, seqs, add):
        page, was = self.page, list(self.ref)
        free = [p for p, r in enumerate(was) if r == 0]
        plans, total, answers = [], 0, []
        for i, (s, x) in enumerate(zip(seqs, add)):
            need, cow = [], None
            bad = not 0 <= s < self.slots or s in seqs[:i] or x < 0
            if not bad:
                want = -(-(self.length[s] + x) // page)
                bad = want > self.width
                at = self.length[s] // page
                if not bad and x > 0 and self.length[s] % page and was[self.table[s][at]] > 1:
                    cow = self.table[s][at]
                grow = 0 if bad else max(0, want - self.held[s])
            n = 0 if bad else grow + (cow is not None)
            total += n
            ok = not bad and (n == 0 or total <= len(free))
            answers.append(int(ok))
            if ok and n:
                plans.append((s, cow, free[total - n:total]))
        for s, cow, got in plans:
            for p in got:
                self.ref[p] = 1
            if cow is not None:
                to, got = got[0], got[1:]
                r = self.length[s] % page
                self.k[:, to, :, :r] = self.k[:, cow, :, :r]
                self.v[:, to, :, :r] = self.v[:, cow, :, :r]
                self.table[s][self.length[s] // page] = to
                self.ref[cow] -= 1
            for p in got:
                self.table[s][self.held[s]] = p
                self.held[s] += 1
        return answers

    def fork(self, parents, children):
        was_held, was_len = list(self.held), list(self.length)
        answers = []
        for i, (p, c) in enumerate(zip(parents, children)):
            ok = 0 <= p < self.slots and 0 <= c < self.slots and c not in children[:i] and p not in children
            ok = ok and was_held[c] == 0 and was_len[c] == 0
            answers.append(int(ok))
            if ok:
                n = -(-self.length[p] // self.page)
                self.table[c][:n] = self.table[p][:n]
                for x in self.table[p][:n]:
                    self.ref[x] += 1
                self.length[c], self.held[c] = self.length[p], n
        return answers

    def release(self, seqs, lengths=None):
        for i, s in enumerate(seqs):
            if not 0 <= s < self.slots or s in seqs[:i]:
                continue
            n = min(self.length[s], max(0, lengths[i]) if lengths is not None else 0)
            keep = -(-n // self.page)
            for j in range(keep, self.held[s]):
                self.ref[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.length[s], self.held[s] = n, keep

    def place(self, s, pos):
        return (self.table[s][pos // self.page], pos % self.page) if 0 <= pos < self.held[s] * self.page else None

    def append(self, layer, k, v, seqs, cu):
        for b, s in enumerate(seqs):
            if not 0 <= s < self.slots:
                continue
            for t in range(cu[b], cu[b + 1]):
                at = self.place(s, self.length[s] + t - cu[b])
                if at is None:
                    continue
                if layer is None:
                    self.k[:, at[0], :, at[1]], self.v[:, at[0], :, at[1]] = k[:, t], v[:, t]
                else:
                    self.k[layer, at[0], :, at[1]], self.v[layer, at[0], :, at[1]] = k[t], v[t]

    def accept(self, seqs, count, path=None, length=None):
        out = self.length if length is None else length
        new = {}
        for i, s in enumerate(seqs):
            if not 0 <= s < self.slots:
                continue
            n = max(0, count[i]) if path is None else min(max(0, count[i]), len(path[i]))
            if path is not None:
                kk, vv = self.k.clone(), self.v.clone()
                for j in range(n):
                    a, b = self.place(s, self.length[s] + path[i][j]) if path[i][j] >= 0 else None, self.place(s, self.length[s] + j)
                    if a and b:
                        self.k[:, b[0], :, b[1]], self.v[:, b[0], :, b[1]] = kk[:, a[0], :, a[1]], vv[:, a[0], :, a[1]]
            new[s] = max(self.length[s], min(self.length[s] + n, self.held[s] * self.page))
        for s, n in new.items():
            out[s] = n

    def same(self, values=True):
        c = self.c
        for name in ("table", "length", "held", "ref"):
            assert getattr(c, name).tolist() == getattr(self, name), name
        if values:  # bits, so that a NaN equals itself
            assert torch.equal(c.k.view(torch.int16), self.k.view(torch.int16)) and torch.equal(c.v.view(torch.int16), self.v.view(torch.int16))

    def tokens(self, layer, s, n):
        """k, v [n][kv heads][d] of a slot's first n tokens"""
        at = [self.place(s, i) for i in range(n)]
        pg, off = [a[0] for a in at], [a[1] for a in at]
        return self.k[layer].transpose(1, 2)[pg, off], self.v[layer].transpose(1, 2)[pg, off]
