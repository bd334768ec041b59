"""How many bits the attention keeps of fp32 queries and of its probabilities: bounds that a
16-bit part less would break, which the 64-bit formula with such parts shows."""
from __future__ import annotations

import pytest
import torch

from test_gpu_step import U, Case

pytestmark = pytest.mark.gpu

# (tokens, query heads, kv heads: up to 16, 32 and 64 rows to a tile)
ROWS = [(3, 4, 2), (7, 8, 2), (19, 8, 2)]
LEAST = {torch.float16: 1, torch.bfloat16: 2}  # one part less than the kernel's


def cut(x, cache):
    """x in so many parts of the cache's type as LEAST has, as the kernel splits it: to
    nearest in fp16, truncated in bf16."""
    rest, out = x.float(), torch.zeros_like(x, dtype=torch.float64)
    for _ in range(LEAST[cache]):
        part = rest.half().float() if cache == torch.float16 else (rest.view(torch.int32) & -65536).view(torch.float32)
        out += part.double()
        rest = rest - part
    return out


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new, hq, hkv", ROWS)
def test_queries_keep_their_bits(D, cache, new, hq, hkv):
    # One key for each of a query's elements, 32 times it: scores of 4 (scale 1/8), of which the
    # even ones are larger by what ends in eight bits that one part less leaves out
    # (2^-15 of them), and values of 1 and -1 by turns.  A score's products are exact; its
    # scale, its reference's subtraction (at most 5.9 in powers of 2) and the
    # exponential are off by 16 U, the sums by 32 + D / 16.
    c = Case([D], [new], hq, hkv, D, cache=cache, tree=True, seed=1)
    c.masks[:] = 0
    even = torch.arange(D) % 2 == 0
    c.q = (1.0 + (255 if cache == torch.float16 else 65535) * 2.0 ** -23 * even).expand(new, hq, D).contiguous()
    for j in range(D):
        p = int(c.table[0, j // 16])
        c.k[p, j % 16] = 32.0 * (torch.arange(D) == j)
        c.v[p, j % 16] = 1.0 if j % 2 == 0 else -1.0
    sign = torch.where(even, 1.0, -1.0).double()

    def formula(q):
        return (torch.softmax(4.0 * q.double(), -1) * sign).sum(-1)
    want, tol = formula(c.q)[..., None], (64 + D / 16) * U
    assert bool(((formula(cut(c.q, cache))[..., None] - want).abs() > 4 * tol).all())
    assert float((c.run(max_new=new, scale=0.125).double().cpu() - want).abs().max()) <= tol


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new, hq, hkv", ROWS)
@pytest.mark.parametrize("length", [60, 250])
def test_probabilities_keep_their_bits(D, cache, new, hq, hkv, length):
    # values of 1: the probabilities' parts against their sum, off by the keys' sums
    c = Case([length], [new], hq, hkv, D, cache=cache, tree=True, seed=2, spread=1.0)
    c.v[torch.isfinite(c.v)] = 1.0
    tol = (32 + (length + new) / 16) * U
    keys = torch.cat([c.k[p] for p in c.table[0, :-(-length // 16)].tolist()])[:length].double()
    s = (c.q.double().view(new, hkv, -1, D) * D ** -0.5) @ keys.permute(1, 2, 0)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    assert float((cut(p, cache).sum(-1) / p.sum(-1) - 1).abs().max()) > 2 * tol
    assert float((c.run(max_new=new).double().cpu() - 1).abs().max()) <= tol
