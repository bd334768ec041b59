"""Caches of 8 bits on the GPU: what qk_norm_rope writes, read_cache reads and keep_accepted
moves, against plain 64-bit implementations."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import step8_ref
import step_ref
from forge_amd import step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # unit roundoff of fp32
G = 16


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache_of(nb, bs, hkv, D, seed, by_head=True):
    """A pair of Cache8 of random codes and scales."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for c in step.paged_cache(nb, bs, hkv, D, torch.int8):
        data = c.codes if by_head else c.codes.contiguous()
        data.copy_(torch.randint(-127, 128, data.shape, generator=g, dtype=torch.int8))
        c.scales.copy_(0.01 * (0.5 + torch.rand(c.scales.shape, generator=g)))
        out.append(step.Cache8(data, c.scales))
    return out


def by_groups(c):
    """Codes [blocks * groups, heads, 16, D] and scales [blocks * groups, heads] of a Cache8, in 64 bits."""
    nb, bs, hkv, D = c.codes.shape
    codes = c.codes.cpu().double().view(nb, bs // G, G, hkv, D).permute(0, 1, 3, 2, 4).reshape(-1, hkv, G, D).numpy().copy()
    return codes, c.scales.cpu().double().transpose(1, 2).reshape(-1, hkv).numpy().copy()


def close(got, codes, scales, room):
    """A Cache8 against groups in 64 bits.  room [groups, heads, 16, D]: how far the rounded value
    may be off, in codes: a code differs only where the value lies so near a border."""
    nb, bs, hkv, D = got.codes.shape
    c, s = by_groups(got)
    # (a scale: the largest's error, its division's and the largest's own rounding)
    assert (np.abs(s - scales) <= scales * 64 * U + 1e-44).all()
    d = np.abs(c - codes)
    assert (d <= room).all(), float((d - room).max())


class Rope:
    def __init__(self, lengths, new, hq, hkv, D, rot, *, bs=16, seed=0, inter=False, bias=False, norm=False,
                 by_head=True, pad=0, scale=1.0, shuffle=True):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.lengths, self.new, self.shape = lengths, new, (hq, hkv, D, rot)
        need = [-(-(a + b) // bs) for a, b in zip(lengths, new)]
        nb = sum(need) + 2
        ids = rng.permutation(nb) if shuffle else np.arange(nb)
        self.caches = cache_of(nb, bs, hkv, D, seed + 1, by_head)
        self.before = [by_groups(c) for c in self.caches]
        self.slots, self.positions, at = [], [], 0
        for a, b, n in zip(lengths, new, need):
            for t in range(a, a + b):
                self.slots.append(int(ids[at + t // bs]) * bs + t % bs)
                self.positions.append(t % 50)
            at += n
        self.N = sum(new)
        width = (hq + 2 * hkv) * D
        self.x = (scale * torch.randn((self.N, width + pad), generator=g)).cuda()[:, :width]
        self.table = step.rope_table(50, rot)
        self.bias = torch.randn(width, generator=g).cuda() if bias else None
        self.qw, self.kw = ((1 + torch.randn(D, generator=g)).cuda() for _ in range(2)) if norm else (None, None)
        self.inter, self.bs = inter, bs

    def run(self):
        return step.qk_norm_rope(self.x, ints(self.positions), ints(self.slots), self.table, *self.caches,
                                 bias=self.bias, q_weight=self.qw, k_weight=self.kw, eps=1e-5, interleaved=self.inter)

    def check(self):
        hq, hkv, D, rot = self.shape
        q = self.run().double().cpu().numpy()

        def np_(v):
            return None if v is None else v.cpu().numpy()
        h = step_ref.norm_rope(np_(self.x), hq, hkv, D, rot, self.inter, np_(self.bias), np_(self.qw), np_(self.kw),
                               1e-5, self.positions, np_(self.table))
        # a rotated element: a norm's factor (D / 8 + 8 roundings) times a sum of two products (3)
        length = np.sqrt((h ** 2).sum(-1, keepdims=True))
        tol = (D / 8 + 16) * U * length + 1e-37
        ok = ~np.isnan(h[:, :hq])
        assert (np.isnan(q) == ~ok).all()
        assert (np.abs(q - h[:, :hq])[ok] <= np.broadcast_to(tol[:, :hq], q.shape)[ok]).all()
        for w, (cache, (codes, scales)) in enumerate(zip(self.caches, self.before)):
            room, first_codes = np.zeros_like(codes), codes.copy()
            rows = h[:, hq + w * hkv:hq + (w + 1) * hkv]
            off = tol[:, hq + w * hkv:hq + (w + 1) * hkv]
            n = 0
            while n < self.N:
                slot, m = self.slots[n], 1
                if slot < 0 or slot // self.bs >= len(cache.codes):
                    n += 1
                    continue
                while n + m < self.N and self.slots[n + m] == slot + m and (slot + m) % G:
                    m += 1
                g, first = slot // G, slot % G
                for k in range(hkv):
                    x = rows[n:n + m, k]
                    fine = np.where(np.isfinite(x), np.abs(x), 0.0)
                    before = float(scales[g, k])
                    most = fine.max()
                    x = np.where(np.isnan(x), 0.0, np.clip(x, -most, most))
                    step8_ref.enter(codes[:, k], scales[:, k], [(g, first, x, most / 127)])
                    s = scales[g, k]
                    if s > 0:
                        # the value's error, the scale's and the product's in codes of up to 127, and half
                        # a code where that reaches a border: then one more code
                        e = np.broadcast_to(off[n:n + m, k], x.shape) / s + 127 * 8 * U
                        near = np.abs(np.abs(x / s - np.floor(x / s)) - 0.5) <= e
                        room[g, k, first:first + m] = near
                        if first and s > before:
                            y = first_codes[g, k, :first] * (before / s)
                            # (the new scale is off by the value's error)
                            e = 127 * (off[n:n + m, k].max() / (127 * s) + 8 * U)
                            room[g, k, :first] = np.abs(np.abs(y - np.floor(y)) - 0.5) <= e
                n += m
            close(cache, codes, scales, room)


@pytest.mark.parametrize("D, rot", [(16, 16), (64, 64), (64, 32), (80, 80), (96, 96), (96, 48), (128, 128), (128, 0),
                                    (256, 256), (256, 64), (512, 512)])
@pytest.mark.parametrize("inter", [False, True])
def test_write(D, rot, inter):
    for i, (bias, norm) in enumerate(((False, False), (True, False), (False, True), (True, True))):
        Rope([5, 0, 31], [3, 40, 2], 6, 2, D, rot, inter=inter, bias=bias, norm=norm, seed=i).check()


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 47])
@pytest.mark.parametrize("new", [1, 2, 15, 16, 17, 33, 100])
def test_write_lengths(length, new):
    Rope([length], [new], 4, 2, 64, 64, seed=length + new, bs=16).check()
    Rope([length, 3, length], [new, 1, new], 3, 1, 128, 128, norm=True, seed=length + new, bs=64).check()


@pytest.mark.parametrize("hq, hkv", [(1, 1), (7, 1), (32, 4), (28, 4), (12, 12)])
def test_write_heads(hq, hkv):
    rng = np.random.default_rng(hq)
    Rope(rng.integers(0, 40, 19).tolist(), [1] * 19, hq, hkv, 64, 64, seed=hq, bs=32).check()
    Rope([9, 100], [300, 31], hq, hkv, 128, 128, seed=hq, bs=128, norm=True).check()


def test_write_strides_layouts_and_missing_slots():
    for by_head in (False, True):
        for pad in (1, 4, 640):
            Rope([5, 3], [20, 9], 4, 2, 64, 64, pad=pad, by_head=by_head, norm=True).check()
    c = Rope([3], [30], 4, 2, 128, 128)
    for i, bad in ((0, -1), (12, -7), (13, 10 ** 9), (28, 2 ** 31 - 1), (29, -2 ** 31)):
        c.slots[i] = bad  # (at groups' ends: what follows the first ones enters a group that holds tokens)
    c.check()
    c = Rope([3], [6], 4, 2, 128, 128, norm=True)
    c.positions = [0, -1, 49, 50, 2 ** 31 - 1, -2 ** 31]  # NaN keys: codes 0
    c.check()


def test_write_blocks_in_order_that_run_on():
    # the last slot of a block and the first of the next are neighbours, of different groups
    Rope([30, 0], [40, 20], 4, 2, 64, 64, bs=32, shuffle=False).check()


@pytest.mark.parametrize("scale", [1e-30, 1e-38, 1e-44, 1e30, 1e37])
def test_write_extremes(scale):
    Rope([4, 0], [9, 33], 4, 2, 64, 64, scale=scale, seed=1).check()


def test_write_zeros_infinities_and_nan():
    c = Rope([0, 20], [20, 5], 2, 1, 64, 64, seed=2)
    c.table = step.rope_table(50, 0)
    c.shape = (2, 1, 64, 0)
    c.x[:16] = 0.0             # a group of zeros
    c.x[17, 3 * 64 + 5] = math.inf
    c.x[18, 2 * 64 + 7] = -math.inf
    c.x[19, 3 * 64 + 1] = math.nan
    c.check()
    k, v = c.caches
    page, row = c.slots[0] // 16, c.slots[17] % 16
    assert not k.codes[page].any() and not k.scales[page].any()
    assert int(v.codes[c.slots[17] // 16, row, 0, 5]) == 127 and int(v.codes[c.slots[19] // 16, c.slots[19] % 16, 0, 1]) == 0
    assert int(k.codes[c.slots[18] // 16, c.slots[18] % 16, 0, 7]) == -127
    only = Rope([0], [4], 2, 1, 64, 64, seed=3)
    only.x[:] = math.inf
    only.run()
    assert not only.caches[1].codes[only.slots[0] // 16, :4].any() and not only.caches[1].scales[only.slots[0] // 16].any()


def test_write_token_by_token_stays_near():
    # sixteen tokens one by one: each rounding of what is held adds half a code at most
    c = Rope([0], [16], 4, 2, 64, 64, seed=4)
    want = step_ref.norm_rope(c.x.cpu().numpy(), 4, 2, 64, 64, False, None, None, None, 1e-5, c.positions, c.table.cpu().numpy())
    for n in range(16):
        step.qk_norm_rope(c.x[n:n + 1], ints(c.positions[n:n + 1]), ints(c.slots[n:n + 1]), c.table, *c.caches)
    page = c.slots[0] // 16
    for w, cache in enumerate(c.caches):
        rows = want[:, 4 + 2 * w:6 + 2 * w]
        got = step8_ref.values(cache.codes[page:page + 1].cpu(), cache.scales[page:page + 1].cpu())[0].numpy()
        most = np.abs(rows).max(-1)  # [16, heads]
        s = most.max(0) / 127
        assert np.allclose(cache.scales[page, :, 0].cpu().numpy(), s, rtol=1e-5)
        grown = np.array([[(np.diff(np.maximum.accumulate(most[:, h])[n:]) > 0).sum() for h in range(2)] for n in range(16)])
        assert (np.abs(got - rows) <= s[None, :, None] * (0.5 * (1 + grown[..., None]) + 1e-3)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv, D", [(1, 16), (4, 64), (3, 96), (2, 512), (8, 128)])
def test_read(dtype, hkv, D):
    for by_head in (True, False):
        bs, lengths = 32, [5, 0, 100, 32, 1]
        k, v = cache_of(12, bs, hkv, D, 7, by_head)
        table = torch.full((5, 6), -1, dtype=torch.int32)
        ids = np.random.default_rng(1).permutation(12)
        at = 0
        for b, n in enumerate(lengths):
            for c in range(-(-n // bs)):
                table[b, c] = int(ids[at])
                at += 1
        table[2, 1] = 12  # no block
        for scales, bad in ((k.scales, math.nan), (v.scales, -1.0)):
            scales[int(table[2, 0])] = bad  # count as 0
        starts = [0] + np.cumsum(lengths).tolist()
        for first, rows in ((None, starts), ([0, 0, 33, 30, 0], [0, 5, 5, 72, 74, 75]), ([-3, 1, 2 ** 31 - 1, 0, 0], starts)):
            N = rows[-1] + 3
            got = step.read_cache(k, v, table.cuda()[:, :5], ints(rows), N, dtype=dtype,
                                  first=None if first is None else ints(first))
            for w, cache in zip(got, (k, v)):
                x = step8_ref.values(cache.codes.cpu(), cache.scales.cpu())
                want = torch.zeros((N, hkv, D), dtype=torch.float64)
                for b in range(5):
                    for i in range(rows[b + 1] - rows[b]):
                        n = (first[b] if first else 0) + i
                        p = int(table[b, n // bs]) if 0 <= n < 5 * bs else -1
                        if 0 <= p < 12:
                            want[rows[b] + i] = x[p, n % bs]
                assert w.dtype == dtype and w.shape == want.shape
                # a product in fp32, rounded once more
                half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}[dtype]
                tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
                assert bool(((w.cpu().double() - want).abs() <= want.abs() * (half + 2 * U) + tiny).all())


def test_read_many_requests_and_none():
    k, v = cache_of(700, 16, 1, 64, 3)
    lengths = np.random.default_rng(2).integers(0, 17, 700)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    kk, vv = step.read_cache(k, v, ints([[b] for b in range(700)]), ints(starts.tolist()), int(starts[-1]), dtype=torch.float32)
    want = torch.cat([step8_ref.values(v.codes[b:b + 1].cpu(), v.scales[b:b + 1].cpu())[0, :n] for b, n in enumerate(lengths)])
    assert bool(((vv.cpu().double() - want).abs() <= want.abs() * 2 * U).all())
    kk, vv = step.read_cache(k, v, ints([[0]]), ints([0, 0]), 0)
    assert kk.shape == (0, 1, 64)


# ---------------------------------------------------------------- accepted branches

class Keep:
    def __init__(self, lengths, new, paths, hkv, D, *, cache=torch.int8, bs=16, seed=0, by_head=True):
        rng = np.random.default_rng(seed)
        self.lengths, self.new, self.bs = lengths, new, bs
        need = [-(-(a + b) // bs) for a, b in zip(lengths, new)]
        nb = sum(need) + 2
        ids, at = rng.permutation(nb), 0
        self.table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            self.table[b, :n] = torch.from_numpy(ids[at:at + n].astype(np.int32))
            at += n
        if cache == torch.int8:
            self.caches = cache_of(nb, bs, hkv, D, seed, by_head)
        else:
            g = torch.Generator().manual_seed(seed)
            self.caches = [c if by_head else c.contiguous() for c in step.paged_cache(nb, bs, hkv, D, cache)]
            for c in self.caches:
                c.copy_(torch.randn(c.shape, generator=g))
        self.cu = [0] + np.cumsum(new).tolist()
        self.path = []
        for n, p in zip(new, paths):
            self.path += p + [-1] * (n - len(p))
        self.accepted = [len(p) for p in paths]

    def place(self, b, n):
        c = n // self.bs
        p = int(self.table[b, c]) if 0 <= n and c < self.table.shape[1] else -1
        return p * self.bs + n % self.bs if 0 <= p < len(self.data(0)) else -1

    def data(self, w):
        c = self.caches[w]
        return c.codes if isinstance(c, step.Cache8) else c

    def moves(self):
        for b in range(len(self.new)):
            t0, out = self.cu[b], []
            for d in range(min(self.accepted[b], self.new[b], 64)):
                p = self.path[t0 + d]
                if p != d and 0 <= p < self.new[b]:
                    src, dst = self.place(b, self.lengths[b] + p), self.place(b, self.lengths[b] + d)
                    if src >= 0 and dst >= 0:
                        out.append((src, dst))
            yield out

    def run(self):
        step.keep_accepted(*self.caches, self.table.cuda(), ints(self.lengths), ints(self.cu), ints(self.path), ints(self.accepted))

    def check(self):
        if not isinstance(self.caches[0], step.Cache8):
            want = []
            for c in self.caches:
                flat = c.cpu().flatten(0, 1).clone()
                old = flat.clone()
                for m in self.moves():
                    for a, z in m:
                        flat[z] = old[a]
                want.append(flat.view(c.shape))
            self.run()
            assert all(torch.equal(c.cpu(), w) for c, w in zip(self.caches, want))
            return
        want = []
        for c in self.caches:
            codes, scales = by_groups(c)
            old, olds = codes.copy(), scales.copy()
            room = np.zeros_like(codes)
            for m in self.moves():
                for k in range(codes.shape[1]):
                    for g in sorted({z // G for _, z in m}):
                        mine = [(a, z) for a, z in m if z // G == g]
                        x = np.stack([old[a // G, k, a % G] * olds[a // G, k] for a, _ in mine])
                        step8_ref.enter(codes[:, k], scales[:, k], [(g, mine[0][1] % G, x, np.abs(x).max() / 127)])
                        s = scales[g, k]
                        # products and the scale's inverse: a few roundings of codes up to 127
                        near = lambda y: np.abs(np.abs(y - np.floor(y)) - 0.5) <= 127 * 8 * U  # noqa: E731
                        h = mine[0][1] % G
                        room[g, k, h:h + len(x)] = near(x / s)
                        if h and s > olds[g, k]:
                            room[g, k, :h] = near(old[g, k, :h] * (olds[g, k] / s))
            want.append((codes, scales, room))
        self.run()
        for c, w in zip(self.caches, want):
            close(c, *w)


TREES = ([[0, 2, 3, 7], [0], [0, 1, 5]], [[0, 4], [0, 1, 2, 3], [0, 24]])


@pytest.mark.parametrize("cache", [torch.int8, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hkv, D", [(1, 16), (4, 64), (2, 96), (8, 128), (2, 256), (1, 512)])
def test_keep(cache, hkv, D):
    for i, paths in enumerate(TREES):
        for by_head in (True, False):
            Keep([0, 14, 37], [8, 4, 25], paths, hkv, D, cache=cache, seed=i, by_head=by_head, bs=16 << i).check()


@pytest.mark.parametrize("cache", [torch.int8, torch.bfloat16])
@pytest.mark.parametrize("length", [0, 1, 9, 15, 16, 31, 100])
def test_keep_lengths(cache, length):
    # from one group into the one before, and over three of them
    Keep([length], [64], [[0] + list(range(5, 64, 2))], 2, 64, cache=cache, seed=length).check()
    Keep([length], [64], [list(range(1, 64))], 2, 128, cache=cache, seed=length).check()
    Keep([length], [64], [[0, 63]], 2, 128, cache=cache, seed=length, bs=64).check()


@pytest.mark.parametrize("cache", [torch.int8, torch.float16])
def test_keep_leaves_the_rest(cache):
    # chains, nothing accepted, requests without tokens, more accepted than there are
    c = Keep([5, 7, 9, 3], [6, 4, 0, 90], [[0, 1, 2, 3], [], [], list(range(80))], 2, 64, cache=cache)
    before = [x.clone() for x in (c.data(0), c.data(1))]
    c.run()
    assert torch.equal(before[0], c.data(0)) and torch.equal(before[1], c.data(1))
    c = Keep([5, 30], [6, 70], [[0, 9, -4, 2 ** 31 - 1, 6], list(range(0, 70, 2))], 2, 64, cache=cache)
    c.accepted = [5, 2 ** 31 - 1]
    c.path = [p if p >= 0 else 3000 for p in c.path]
    c.check()
    c = Keep([5, 30], [6, 20], [[0, 4], [0, 5, 19]], 2, 64, cache=cache)
    c.table[0, 0], c.table[1, 3] = -1, 10 ** 6  # no blocks
    c.check()
    c = Keep([5], [6], [[0, 4]], 2, 64, cache=cache)
    c.lengths = [2 ** 31 - 3]
    c.check()


def test_refusals():
    k, v = cache_of(3, 16, 2, 64, 1)
    t, x, p = ints([[0, 1]]), torch.zeros((1, 4 * 64 + 2 * 2 * 64), device="cuda"), ints([0])
    q, table = torch.zeros((1, 4, 64), device="cuda"), step.rope_table(4, 64)
    half = k.codes.half()
    for bad, match in (
            (lambda: step.qk_norm_rope(x, p, p, table, k.codes, v.codes), "fp16 or bf16"),
            (lambda: step.qk_norm_rope(x, p, p, table, k, v.codes), "must be a tensor"),
            (lambda: step.qk_norm_rope(x, p, p, table, step.Cache8(half, k.scales), step.Cache8(half, v.scales)), "int8"),
            (lambda: step.qk_norm_rope(x, p, p, table, step.Cache8(k.codes, k.scales[:2]), v), "scales"),
            (lambda: step.qk_norm_rope(x, p, p, table, step.Cache8(k.codes, k.scales.double()), v), "scales"),
            (lambda: step.qk_norm_rope(x, p, p, table, (k.codes, k.scales, 1), v), "codes, scales"),
            (lambda: step.read_cache(half, half, t, ints([0, 1]), 1), "Cache8"),
            (lambda: step.read_cache(k, v, t, ints([0, 1]), 1, dtype=torch.int8), "dtype"),
            (lambda: step.read_cache(k, v, t, ints([0]), 1), "starts"),
            (lambda: step.read_cache(k, v, t, ints([0, 1]), -1), "n_tokens"),
            (lambda: step.read_cache(k, v, t, ints([0, 1]), 1, first=ints([0, 0])), "first"),
            (lambda: step.read_cache(k, v, ints([[0], [1]]), ints([0, 1]), 1), "block_table"),
            (lambda: step.tree_attention(q, k, v, t, p, ints([0, 1]), window=0), "window"),
            (lambda: step.tree_attention(q, k, v, t, p, ints([0, 1]), window=4, sinks=-1), "sinks"),
            (lambda: step.tree_attention(q, k, v, t, p, ints([0, 1]), sinks=1), "sinks"),
            (lambda: step.keep_accepted(k, v, t, p, ints([0, 1]), p.long(), p), "path"),
            (lambda: step.keep_accepted(k, v, t, p, ints([0, 1]), p, ints([0, 1])), "accepted"),
            (lambda: step.keep_accepted(k, v.codes, t, p, ints([0, 1]), p, p), "must be a tensor")):
        with pytest.raises(RuntimeError, match=match):
            bad()
