"""The check of attention over long contexts sees the mistakes that a split over many blocks can make (CPU only: the mistakes are
planted in the outputs that the 64-bit form gives on changed inputs)."""
import pytest
import torch

import attention_ref as ref
from long_context import values

BF, F16 = torch.bfloat16, torch.float16


def drop(first, n):
    return lambda k, v: (torch.cat([k[:first], k[first + n:]]), torch.cat([v[:first], v[first + n:]]))


def repeat(first, n):
    return lambda k, v: (torch.cat([k[:first + n], k[first:]]), torch.cat([v[:first + n], v[first:]]))


def zeroed(first, n):
    def f(k, v):
        v = v.clone()
        v[first:first + n] = 0
        return k, v
    return f


def off(first, n, by):
    def f(k, v):
        v = v.clone()
        v[first:first + n] = v[first + by:first + by + n].clone()
        return k, v
    return f


def swapped(a, b, n):
    def f(k, v):
        v = v.clone()
        v[a:a + n], v[b:b + n] = v[b:b + n].clone(), v[a:a + n].clone()
        return k, v
    return f


FAULTS = {"two units left out": drop(12800, 256), "a unit left out": drop(1280, 128), "a unit twice": repeat(640, 128),
          "a unit's values zero": zeroed(6400, 128), "2048 values one page of 64 off": off(4096, 2048, 64),
          "2048 values one chunk off": off(4096, 2048, 16), "units in each other's place": swapped(2560, 5120, 128),
          "the last unit left out": drop(19968, 33), "the first left out": drop(0, 128)}


@pytest.mark.parametrize("n,d,dtype", [(70001, 128, BF), (70001, 64, BF), (70001, 256, BF), (20001, 128, F16), (20001, 256, F16)])
def test_the_check_sees(n, d, dtype):
    g = torch.Generator()
    g.manual_seed(d)
    q, k = torch.randn(2, d, generator=g).to(dtype), torch.randn(n, d, generator=g).to(dtype)
    v = values(n, d, dtype)
    all_seen = lambda x: torch.ones(2, len(x), dtype=torch.bool)
    o, l, ob, lb = ref.rows(q, k, v, all_seen(k), d ** -0.5)
    ref.check(o.to(dtype), l.float(), o, l, ob, lb)
    for name, fault in FAULTS.items():
        if dtype is F16 and name == "units in each other's place":
            continue  # columns keep their values, only weights change: less than the bound's n 2^-25 of fp16 probabilities
        fk, fv = fault(k, v)
        wrong = ref.rows(q, fk, fv, all_seen(fk), d ** -0.5)[0]
        with pytest.raises(AssertionError, match="off by"):
            ref.check(wrong.to(dtype), None, o, None, ob, None)
            pytest.fail(f"not seen: {name}")
