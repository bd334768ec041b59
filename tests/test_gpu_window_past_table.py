"""Windows over requests whose length reaches, or passes, the block table's columns: a token's
position is its length + depth all the same, keys past the columns are not there, and a token that
sees none has zeros."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import step8_ref
from forge_amd import _lib, step
from test_gpu_step import tree_masks

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # unit roundoff of fp32
TYPES = {torch.int8: 101, torch.float16: 1, torch.bfloat16: 100}
INT_MAX = 2 ** 31 - 1


def sees(length, n, masks, window, sinks, cap):
    """[n, cap]: which of the table's keys the new tokens of one request see."""
    j = np.arange(cap)
    see = np.zeros((n, cap), dtype=bool)
    for i in range(n):
        bits = list(range(i + 1)) if masks is None else [t for t in range(min(n, 64)) if masks[i] >> t & 1]
        depth = i if masks is None else max(bin(masks[i] % 2 ** 64).count("1") - 1, 0)
        see[i] = (j < length) & ((length + depth - j < window) | (j < sinks))
        for below, t in enumerate(bits):  # (a new key's position: how many bits of the mask lie below)
            if length + t < cap and (depth - below < window or length + below < sinks):
                see[i, length + t] = True
    return see


def check(cache, lengths, new, cap, window, sinks, *, tree=False, hq=4, hkv=2, D=64, bs=16, seed=0):
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    B, cols, cu = len(new), cap // bs, [0] + np.cumsum(new).tolist()
    N, nb = cu[-1], B * cols
    table = torch.from_numpy(rng.permutation(nb).astype(np.int32)).view(B, cols)
    masks = tree_masks(rng, new) if tree else None
    pair, values = [], []
    for _ in range(2):
        if cache == torch.int8:
            codes = torch.randint(-127, 128, (nb, bs, hkv, D), generator=g, dtype=torch.int8)
            scales = 0.02 * torch.exp2(torch.randn((nb, hkv, bs // 16), generator=g))
            pair += [codes.cuda(), scales.cuda()]
            values.append(step8_ref.values(codes, scales))
        else:
            x = torch.randn((nb, bs, hkv, D), generator=g).to(cache)
            pair += [x.cuda(), None]
            values.append(x.double())
    q = (0.4 if cache == torch.int8 else 2.0) * torch.randn((N, hq, D), generator=g)
    scale = D ** -0.5
    dev = dict(dtype=torch.int32, device="cuda")
    ln, cud, dq, dt = torch.tensor(lengths, **dev), torch.tensor(cu, **dev), q.cuda(), table.cuda()
    dm = None if masks is None else torch.tensor(masks, dtype=torch.int64, device="cuda")
    out = torch.full((N, hq, D), math.nan, device="cuda")  # (what is not written stays NaN)
    k, ks, v, vs = pair
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    _lib.check(_lib.lib().fq_window_attention(
        p(dq), hq * D, p(ln), p(cud), p(dm), B, N, max(new), hq, hkv, D, scale, window, sinks, TYPES[cache], p(k), p(v), p(ks),
        p(vs), nb, bs, k.stride(0), k.stride(1), k.stride(2), p(dt), cols, cols, p(out),
        torch.cuda.current_stream().cuda_stream), "attention")
    got = out.double().cpu()
    # scores are off by 2^-20 of |q| |k| at most, a probability by twice that and by the roundings of
    # its exponential, its parts and the keys' sums
    ds = 2.0 ** -20 * scale * float(q.norm(dim=-1).max()) * float(values[0].norm(dim=-1).max())
    tol = float(values[1].abs().max()) * (2 * ds + (32 + cap / 16) * U)
    for b in range(B):
        at = slice(cu[b], cu[b + 1])
        see = torch.from_numpy(sees(lengths[b], new[b], None if masks is None else masks[at], window, sinks, cap))
        kk, vv = (x[table[b].long()].reshape(cap, hkv, D).repeat_interleave(hq // hkv, 1) for x in values)
        s = torch.stack([q[at].double()[:, h] @ kk[:, h].T for h in range(hq)], 1) * scale  # [n, hq, cap]
        pr = torch.nan_to_num(torch.softmax(s.masked_fill(~see[:, None], -math.inf), -1), 0.0)
        want = torch.stack([pr[:, h] @ vv[:, h] for h in range(hq)], 1)
        none = ~see.any(1)
        assert bool((got[at][none] == 0).all()), (b, "a token that sees nothing")
        assert float((got[at] - want).abs().max()) <= tol, b


WINDOWS = [(1, 0), (1, 3), (2, 0), (5, 0), (33, 0), (60, 20), (100, 0), (200, 130), (INT_MAX, 0)]


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("window, sinks", WINDOWS)
def test_lengths_around_the_columns(cache, tree, window, sinks):
    for length in (126, 127, 128, 129, 133, 160, 400, INT_MAX):
        check(cache, [length], [1], 128, window, sinks, tree=tree)
        check(cache, [50, length, 128], [2, 9, 1], 128, window, sinks, tree=tree, D=128, hq=7, hkv=1, seed=length % 97)


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 8, 40])
def test_of_every_tile_height(cache, D, new):
    for cap in (64, 256, 272):
        check(cache, [cap, cap + 1, cap - 1], [new, 1, new], cap, 1, 0, D=D, hq=8, hkv=2)
        check(cache, [cap, cap + 20, 3], [new, new, new], cap, 30, 2, D=D, hq=8, hkv=2, bs=16, tree=True)


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 200), (700, 0), (3000, 90)])
def test_long_tables(cache, window, sinks):
    """Tables of so many keys that items are shared out among the work-groups."""
    cap = 4096
    check(cache, [cap], [1], cap, window, sinks)
    check(cache, [cap, cap + 500, 2000, cap - 1, INT_MAX - 70], [3, 1, 5, 64, 64], cap, window, sinks, hq=8, hkv=2, D=128, bs=64)
