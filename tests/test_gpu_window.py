"""Attention over caches of 8 bits, and with sliding windows and sinks over caches of any
type, against the plain 64-bit implementation."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import step8_ref
from forge_amd import step
from test_gpu_step import tree_masks

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # unit roundoff of fp32
TYPES = [torch.int8, torch.float16, torch.bfloat16]


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Case:
    """Requests over a cache whose every other value is NaN, in 8 bits with scales of NaN."""

    def __init__(self, lengths, new, hq, hkv, D, *, cache=torch.int8, bs=16, tree=False, seed=0, pad=0, by_head=True,
                 spread=2.0, padding=0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.new, self.D = lengths, new, D
        self.cu = [0] + np.cumsum(new).tolist()
        self.N = self.cu[-1] + padding
        need = [-(-(a + b) // bs) for a, b in zip(lengths, new)]
        nb = sum(need) + 3
        ids = rng.permutation(nb)
        self.table = torch.full((len(new), max(need + [1]) + 2), 2 ** 30, dtype=torch.int32)  # never to be followed
        live = torch.zeros((nb, bs), dtype=torch.bool)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.from_numpy(ids[at:at + n].astype(np.int32))
            for c in range(n):
                live[int(ids[at + c]), :min(bs, lengths[b] + new[b] - c * bs)] = True
            at += n
        self.caches = []
        for _ in range(2):
            if cache == torch.int8:
                codes = torch.randint(-128, 128, (nb, bs, hkv, D), generator=g, dtype=torch.int8)
                scales = 0.02 * torch.exp2(2 * torch.randn((nb, hkv, bs // 16), generator=g))
                scales[~live.view(nb, bs // 16, 16).any(-1)[:, None].expand_as(scales)] = math.nan
                self.caches.append(step.Cache8(codes, scales))
            else:
                x = torch.randn((nb, bs, hkv, D), generator=g).to(cache)
                x[~live] = math.nan
                self.caches.append(x)
        self.q = spread * torch.randn((self.N, hq, D), generator=g)
        if cache == torch.int8:
            self.q *= 0.2
        self.pad, self.by_head, self.masks = pad, by_head, None
        if tree:
            self.masks = torch.tensor(tree_masks(rng, new) + [-1] * padding, dtype=torch.int64)

    def data(self):
        def place(x):
            return x.transpose(1, 2).contiguous().cuda().transpose(1, 2) if self.by_head else x.cuda()
        return [step.Cache8(place(c.codes), c.scales.cuda()) if isinstance(c, step.Cache8) else place(c) for c in self.caches]

    def values(self):
        return [step8_ref.values(*c) if isinstance(c, step.Cache8) else c.double() for c in self.caches]

    def run(self, **kw):
        q = self.q.cuda()
        if self.pad:  # tokens further apart than their heads
            wide = torch.full((self.N, q[0].numel() + self.pad), math.nan, device="cuda")
            wide[:, :q[0].numel()] = q.flatten(1)
            q = wide.as_strided(q.shape, (wide.stride(0), self.D, 1))
        return step.tree_attention(q, *self.data(), self.table.cuda(), ints(self.lengths), ints(self.cu),
                                   None if self.masks is None else self.masks.cuda(), **kw)

    def check(self, **kw):
        out = self.run(**kw).double().cpu()
        k, v = self.values()
        scale = kw.get("scale", self.D ** -0.5)
        want = step8_ref.attention(self.q, k, v, self.table, self.lengths, self.cu,
                                   None if self.masks is None else self.masks.tolist(), scale, kw.get("window") or 0,
                                   kw.get("sinks", 0))
        # a score is a sum of D products of a query of 22 bits and more with a key, held in fp32 or
        # exactly, times scales: off by at most 2^-20 of |q| |k|; a probability by twice that (its own
        # and the sum's) and the exponential's, the parts' and the keys' sums' roundings
        k, v = torch.nan_to_num(k, 0.0), torch.nan_to_num(v, 0.0)
        there = torch.isfinite(self.q).all(-1)  # (rows whose query is finite)
        ds = 2.0 ** -20 * abs(scale) * float(self.q[there].norm(dim=-1).max()) * float(k.norm(dim=-1).max())
        most = max(a + b for a, b in zip(self.lengths, self.new))
        tol = float(v.abs().max()) * (2 * ds + (32 + most / 16) * U)
        assert bool(torch.isfinite(out[there]).all())
        err = float((out - want)[there].abs().max()) if out.numel() else 0.0
        assert err <= tol, (err, tol)
        return out


HEADS = [(1, 1), (4, 1), (7, 1), (8, 2), (6, 6), (28, 4)]


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("hq, hkv", HEADS)
def test_codes_heads(D, hq, hkv):
    Case([37], [1], hq, hkv, D).check()
    Case([0, 130, 5], [3, 9, 6], hq, hkv, D, tree=True, seed=1).check()


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 300, 1025])
@pytest.mark.parametrize("new", [1, 2, 5, 17])
def test_codes_lengths(length, new):
    Case([length], [new], 8, 2, 64, seed=length).check(max_new=new)
    Case([length, 3, length], [new, 1, new], 4, 2, 128, bs=32, tree=True, seed=length).check(max_new=new)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("new", [1, 3, 4, 7, 8, 9, 16, 33, 63, 64])
def test_codes_trees(D, new):
    Case([200, 77], [new, max(1, new // 2)], 8, 2, D, tree=True, seed=new).check(max_new=new)
    Case([90], [new], 7, 1, D, seed=new).check(max_new=new)


@pytest.mark.parametrize("bs", [16, 32, 64, 256, 1024])
def test_codes_block_sizes_layouts_and_strides(bs):
    for by_head in (True, False):
        Case([70, 1100], [5, 2], 8, 4, 64, bs=bs, by_head=by_head, tree=True, pad=12).check()
        Case([70, 33], [5, 2], 8, 4, 128, bs=bs, by_head=by_head, pad=1).check()


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("window", [0, 5, 100])
def test_ragged_batches(cache, window):
    rng = np.random.default_rng(5)
    kw = dict(window=window, sinks=3) if window else {}
    for seed in range(5):
        B = int(rng.integers(2, 40))
        lengths = [int(v) for v in np.where(rng.random(B) < 0.2, 0, rng.integers(0, 400, B))]
        new = [int(v) for v in rng.integers(0, 12, B)]
        new[0] += 1
        out = Case(lengths, new, 6, 2, 64, cache=cache, tree=seed % 2 == 0, seed=seed, padding=seed).check(**kw)
        assert not out[sum(new):].any()


@pytest.mark.parametrize("window", [0, 9])
def test_many_requests(window):
    rng = np.random.default_rng(6)
    kw = dict(window=window, sinks=1) if window else {}
    Case(rng.integers(0, 40, 700).tolist(), rng.integers(0, 3, 700).tolist(), 2, 1, 64, seed=7).check(max_new=2, **kw)


def test_long_context_in_many_parts():
    Case([30011], [3], 4, 1, 64, bs=64, tree=True, seed=8).check(max_new=3)
    Case([9000, 100, 20000], [2, 7, 1], 4, 2, 128, bs=32, seed=9).check()


def test_codes_more_than_64_tokens_of_a_chain():
    Case([50, 0], [70, 131], 4, 2, 64, seed=10).check()
    c = Case([50], [70], 4, 2, 64, seed=10)
    c.masks = torch.tensor([(1 << min(i, 63)) - 1 for i in range(70)], dtype=torch.int64)
    c.check()


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("length", [0, 1, 15, 33, 64, 200, 777])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 1), (2, 5), (15, 4), (16, 0), (17, 16), (64, 4), (100, 40), (2 ** 31 - 1, 0),
                                           (50, 2 ** 31 - 1)])
def test_window(cache, tree, length, window, sinks):
    kw = dict(window=window, sinks=sinks)
    Case([length], [1], 4, 2, 64, cache=cache, seed=length).check(**kw)
    Case([length, 20, length], [6, 1, 19], 4, 2, 128, cache=cache, tree=tree, bs=32, seed=length).check(**kw)


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("hq, hkv", [(1, 1), (7, 1), (8, 2)])
def test_window_heads(cache, D, hq, hkv):
    for new in (1, 3, 9, 40):
        Case([300, 31], [new, 2], hq, hkv, D, cache=cache, tree=new == 9, seed=new).check(window=37, sinks=4)


@pytest.mark.parametrize("cache", TYPES)
def test_window_of_a_long_context(cache):
    Case([20011, 5000], [3, 1], 4, 1, 64, cache=cache, bs=64, tree=True, seed=8).check(window=4096, sinks=4)
    Case([9000, 100, 20000], [2, 7, 1], 4, 2, 128, cache=cache, bs=32, seed=9).check(window=1000, sinks=70)
    Case([700], [300], 4, 2, 64, cache=cache, seed=10).check(window=128, sinks=4)  # a chunk of prompt


@pytest.mark.parametrize("cache", TYPES)
def test_window_drops_old_tokens_of_the_draft(cache):
    # a chain as masks: 40 new tokens, a window of 7 of them; sinks among the new ones
    for length in (0, 2, 50):
        c = Case([length], [40], 4, 2, 64, cache=cache, seed=11)
        chain = c.check(window=7, sinks=3)
        c.masks = torch.tensor([(1 << (i + 1)) - 1 for i in range(40)], dtype=torch.int64)
        assert float((c.check(window=7, sinks=3) - chain).abs().max()) <= 1e-4 * float(chain.abs().max())


@pytest.mark.parametrize("cache", TYPES)
def test_what_no_token_sees_is_not_read(cache):
    # blocks outside window and sinks: no entry, NaN, codes of any kind
    c = Case([1000], [2], 4, 2, 64, cache=cache, seed=12)
    want = c.run(window=50, sinks=4)
    for p in c.table[0, 2:58].tolist():
        for x in c.caches:
            if isinstance(x, step.Cache8):
                x.codes[p], x.scales[p] = 127, math.inf
            else:
                x[p] = math.nan
    assert torch.equal(c.run(window=50, sinks=4), want)
    c.table[0, 2:58] = -1
    assert torch.equal(c.run(window=50, sinks=4), want)


@pytest.mark.parametrize("cache", TYPES)
def test_missing_blocks_and_rows_that_see_nothing(cache):
    c = Case([100, 40], [5, 3], 8, 2, 64, cache=cache, tree=True, seed=13)
    c.table[0, 2], c.table[1, 0] = -1, 2 ** 30
    c.check()
    c.check(window=30, sinks=2)
    c.table[1, :] = -1
    assert not c.check()[5:].any()
    c = Case([0, 0, 40], [4, 1, 3], 8, 2, 64, cache=cache, tree=True, seed=12)
    c.masks[:] = 0
    out = c.check()
    assert not out[:5].any() and out[5:].abs().sum() > 0
    c.masks[1] = 1
    out = c.check()
    assert not out[0].any() and bool(out[1].any())


def test_codes_lengths_past_the_table():
    c = Case([100], [5], 8, 2, 64, seed=14)
    c.table = c.table[:, :3].contiguous()
    c.lengths = [2 ** 31 - 1]  # every key of the three blocks, and no other
    out = c.run().double().cpu()
    k, v = c.values()
    assert bool(torch.isfinite(out).all())
    full = step8_ref.attention(c.q[:1], k, v, c.table, [47], [0, 1], None, 8 ** -1.0)
    assert float((out[0] - full[0]).abs().max()) <= 1e-4 * float(full.abs().max())


def test_codes_scales_that_are_none_count_as_zero():
    for which in range(2):
        for bad in (math.nan, math.inf, -1.0, 0.0, -math.inf):
            c = Case([100], [3], 8, 2, 64, tree=True, seed=15)
            c.caches[which].scales[int(c.table[0, 1])] = bad
            c.caches[which].scales[int(c.table[0, 6])] = bad  # of the new tokens too
            c.check()


def test_codes_scales_far_apart():
    # groups of values 2^-60 and 2^60 of others; a row that sees only small ones keeps its bits
    c = Case([200], [4], 4, 1, 64, tree=True, seed=16)
    c.caches[1].scales[int(c.table[0, 3])] = 2.0 ** 60
    c.caches[1].scales[int(c.table[0, 5])] = 2.0 ** -60
    c.check()
    c = Case([0], [40], 4, 1, 64, tree=True, seed=17)
    c.masks = torch.tensor([1 << i for i in range(40)], dtype=torch.int64)  # each its own key alone
    c.caches[1].scales[int(c.table[0, 0])] = 2.0 ** 60
    c.caches[1].scales[int(c.table[0, 1])] = 2.0 ** -60
    out, v = c.run().double().cpu(), c.values()[1]
    for i in range(40):
        want = v[int(c.table[0, i // 16]), i % 16, 0]
        assert float((out[i] - want).abs().max()) <= 40 * U * float(want.abs().max())
    c = Case([300], [4], 4, 2, 128, seed=18)
    c.caches[0].scales.mul_(2.0 ** -40)
    c.q *= 2.0 ** 40
    c.check()
    Case([300], [4], 4, 2, 128, seed=17).check(scale=-0.3)
    Case([300], [4], 4, 2, 128, seed=17).check(scale=0.0)
    c = Case([300], [4], 4, 2, 128, seed=17)
    c.q[1] = 0.0
    c.check()


@pytest.mark.parametrize("log", [-79, -40, 60, 100, 119])
@pytest.mark.parametrize("D, new", [(64, 3), (128, 20), (256, 9)])
def test_codes_values_of_any_size(log, D, new):
    c = Case([700, 20], [new, 1], 8, 2, D, tree=True, seed=21)
    c.caches[1].scales[:] = 2.0 ** log * (1 + torch.rand(c.caches[1].scales.shape, generator=torch.Generator().manual_seed(1)))
    c.check()
    c.check(window=300, sinks=4)


@pytest.mark.parametrize("log", [61, 90, 118])
@pytest.mark.parametrize("hq, D, new", [(4, 64, 64), (4, 128, 64), (1, 128, 33), (4, 256, 50)])
def test_codes_large_values_behind_small_ones(log, hq, D, new):
    # rows that see small ones alone keep their bits, before and after the first large one
    c = Case([0], [new], hq, 1, D, tree=True, seed=25)
    pages = c.table[0, :-(-new // 16)].tolist()
    for i, p in enumerate(pages):
        c.caches[1].scales[p] = 2.0 ** (log if i == 2 else -6)
    c.masks = torch.tensor([1 << i if i < 63 else -2 ** 63 for i in range(new)], dtype=torch.int64)  # each its own key alone
    out, v = c.run(max_new=new).double().cpu(), c.values()[1]
    for i in range(new):
        want = v[pages[i // 16], i % 16, 0]
        assert float((out[i] - want).abs().max()) <= 40 * U * float(want.abs().max())
    c = Case([100 * 16], [3], hq, 1, D, seed=26)
    for i in (0, 55, 99):  # (what is small vanishes beside it)
        c.caches[1].scales[int(c.table[0, i])] = 2.0 ** log
        c.check()


def test_codes_scores_far_apart():
    for at in (0, 35, 199, 203):
        c = Case([200], [4], 4, 1, 64, seed=15)
        p = int(c.table[0, at // 16])
        c.caches[0].codes[p, at % 16] = (127 * torch.sign(c.q[3, 0])).to(torch.int8)
        c.caches[0].scales[p] = 0.4
        c.check()


def test_queries_keep_their_bits():
    # one key for each of a query's elements: scores of about 4, of which the even ones are larger by
    # 255 2^-23 of that; fp32 keeps it, 16 bits of a query would not
    for D in (64, 96, 128, 256):
        for new, hq, hkv in ((3, 4, 2), (7, 8, 2), (19, 8, 2)):
            c = Case([D], [new], hq, hkv, D, tree=True, seed=1)
            c.masks[:] = 0
            even = torch.arange(D) % 2 == 0
            c.q = (1.0 + 255 * 2.0 ** -23 * even).expand(new, hq, D).contiguous()
            for x in c.caches:
                x.codes[:], x.scales[:] = 0, 0.25
            for j in range(D):
                p = int(c.table[0, j // 16])
                c.caches[0].codes[p, j % 16] = 127 * (torch.arange(D) == j)
                c.caches[1].codes[p, j % 16] = 127 if j % 2 == 0 else -127
            s = c.q.double() * 127 * 0.25 / 8
            want = (torch.softmax(s, -1) * torch.where(even, 1.0, -1.0).double()).sum(-1)[..., None] * 127 * 0.25
            out = c.run(max_new=new, scale=0.125).double().cpu()
            # scores of 4 in powers of two, rounded as above; sums of D values
            assert float((out - want).abs().max()) <= 127 * 0.25 * (64 + D / 16) * U
            assert float(want.abs().max()) > 4 * 127 * 0.25 * (64 + D / 16) * U


def test_probabilities_keep_their_bits():
    # equal values: what the probabilities' parts add up to against their sum
    for D in (64, 128, 256):
        for new, hq, hkv in ((3, 4, 2), (7, 8, 2), (19, 8, 2)):
            c = Case([250], [new], hq, hkv, D, tree=True, seed=2)
            c.caches[1].codes[:], c.caches[1].scales[:] = 64, 2.0 ** -6
            out = c.run(max_new=new).double().cpu()
            assert float((out - 1).abs().max()) <= (32 + (250 + new) / 16) * U


def test_codes_of_a_long_cache_past_32_bit_offsets():
    nb, bs, hkv, D = 82000, 64, 8, 128  # 5 GiB of codes
    caches = []
    for w in range(2):
        codes = torch.empty((nb, hkv, bs, D), dtype=torch.int8, device="cuda").transpose(1, 2)
        codes[:3] = 100
        codes[-3:] = torch.randint(-127, 128, (3, bs, hkv, D), dtype=torch.int8, device="cuda")
        scales = torch.full((nb, hkv, bs // 16), 0.01, device="cuda")
        caches.append(step.Cache8(codes, scales))
    table = ints([[nb - 2, nb - 1, nb - 3]])
    q = 2 * torch.randn((2, 16, D), device="cuda")
    x = torch.randn((2, (16 + 2 * hkv) * D), device="cuda")
    slots = ints([(nb - 3) * 64 + 22, (nb - 3) * 64 + 23])
    step.qk_norm_rope(x, ints([150, 151]), slots, step.rope_table(200, D), *caches)
    small = [step.Cache8(c.codes[-3:].contiguous(), c.scales[-3:].clone()) for c in caches]  # (a slice of scales is contiguous)
    near = ints([[1, 2, 0]])
    for kw in ({}, dict(window=70, sinks=4)):
        a = step.tree_attention(q, *caches, table, ints([150]), ints([0, 2]), **kw)
        assert torch.equal(a, step.tree_attention(q, *small, near, ints([150]), ints([0, 2]), **kw))
    a, b = (step.read_cache(*c, t, ints([0, 152]), 152) for c, t in ((caches, table), (small, near)))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for c, t in ((caches, table), (small, near)):
        step.keep_accepted(*c, t, ints([120]), ints([0, 32]), ints([0, 9, 31] + [-1] * 29), ints([3]))
    assert all(torch.equal(c.codes[-3:], s.codes) and torch.equal(c.scales[-3:], s.scales) for c, s in zip(caches, small))
    assert bool((caches[0].codes[:3] == 100).all())


@pytest.mark.parametrize("cache", TYPES)
def test_max_new_is_only_a_hint(cache):
    c = Case([100, 20], [21, 4], 8, 2, 64, cache=cache, tree=True, seed=11)
    for hint in (0, 1, 4, 21, 64, 10 ** 6):
        c.check(max_new=hint)
        c.check(max_new=hint, window=9, sinks=2)


@pytest.mark.parametrize("window", [None, 33])
def test_results_repeat(window):
    c = Case([9000, 500, 0], [9, 3, 1], 8, 2, 128, tree=True, seed=19)
    first = c.run(window=window)
    assert all(torch.equal(first, c.run(window=window)) for _ in range(3))


@pytest.mark.parametrize("cache", TYPES)
@pytest.mark.parametrize("window", [None, 40])
def test_a_query_that_is_not_finite_is_its_rows_alone(cache, window):
    # (several rows to a lane, several lanes' rows to a tile, two waves' rows to an item)
    for new, hq, hkv, D in ((3, 4, 1, 64), (9, 8, 2, 128), (40, 8, 2, 64), (9, 8, 2, 256)):
        c = Case([150], [new], hq, hkv, D, cache=cache, seed=new)
        want = c.run(window=window)
        c.q[1, 1, 7], c.q[2, 0, 0] = math.nan, math.inf
        out = c.check(window=window)
        assert bool(torch.isnan(out[1, 1]).all())
        if cache == torch.int8:  # (in 16 bits a tile with such a row is summed another way, for all of its rows)
            mine = torch.ones((new, hq), dtype=torch.bool)
            mine[1, 1] = mine[2, 0] = False
            assert torch.equal(out[mine], want.double().cpu()[mine])


@pytest.mark.parametrize("cache", TYPES)
def test_masks_of_no_bits_under_a_window(cache):
    # position len: the last window - 1 cached keys and the sinks
    c = Case([100, 3], [5, 2], 8, 2, 64, cache=cache, tree=True, seed=22)
    c.masks[:] = 0
    for window, sinks in ((1, 0), (2, 0), (30, 5), (1, 2)):
        out = c.check(window=window, sinks=sinks)
        assert bool(out.any()) == (window > 1 or sinks > 0)


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("window", [None, 1500])
def test_codes_every_tile_height(D, window):
    # items of 16 rows, of 32 to 128 and of more, cut and whole
    for lengths, new in (([4000, 300], [1, 2]), ([4000, 2500] * 12, [12, 5] * 12), ([3000] * 16, [40] * 16)):
        Case(lengths, new, 8, 2, D, bs=64, seed=23).check(max_new=max(new), window=window, sinks=4 if window else 0)


@pytest.mark.parametrize("cache", TYPES)
def test_requests_that_share_blocks(cache):
    # the same prefix's blocks in several tables, and a block twice in one
    c = Case([90, 90, 90], [3, 1, 4], 4, 2, 64, cache=cache, seed=24)
    c.table[1, :5] = c.table[0, :5]
    c.table[2, 1] = c.table[2, 0]
    c.check()
    c.check(window=40, sinks=17)
