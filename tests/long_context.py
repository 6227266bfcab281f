"""Values for attention over tens of thousands of tokens on which the error bound of attention_ref.py can fail: of one sign, so
that an output does not average to nearly nothing, and each unit of 128 tokens in a column of its own (modulo the head size), so
that a unit that is left out, repeated or read in another's place shows as a large part of one column. Units and chunks of 16
tokens have values of their own, so that units in each other's place and rows read one page off show too."""
import torch


def values(n, d, dtype, device="cpu"):
    j = torch.arange(n, device=device)
    v = torch.zeros(n, d, device=device)
    mixed = lambda x: x * 2654435761 % 2 ** 32 >> 16
    v[j, j // 128 % d] = 1.0 + 3.0 * (mixed(j // 128) % 3) + mixed(j // 16) % 3
    return v.to(dtype)
