"""The step operators (plan, norm and rotation, tree attention, log probabilities)
on the GPU against their plain 64-bit implementations, over types, head layouts,
lengths from nothing to long, odd sizes, strides, masks that leave a row empty,
NaN and infinities in masked places, other streams and graph replays."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import step_ref
from forge_amd import step

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # unit roundoff of fp32


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan

def random_parents(rng, new, N):
    p = []
    for n in new:
        p += [int(rng.integers(-1, i)) if i else -1 for i in range(max(0, n))]
    return (p + [0] * N)[:N]


def run_plan(lengths, new, parents, cols, bs, N, n_free, seed=0, stride=None):
    rng = np.random.default_rng(seed)
    B = len(lengths)
    ids = rng.permutation(B * cols + n_free + 7).astype(np.int32)
    table = ids[:B * cols].reshape(B, cols)
    free = ids[B * cols:B * cols + n_free]
    wide = torch.full((B, (stride or cols)), -77, dtype=torch.int32, device="cuda")
    wide[:, :cols] = torch.from_numpy(table).cuda()
    got = step.plan_step(ints(lengths), ints(new), wide[:, :cols], torch.from_numpy(free).cuda(), bs, N,
                         parents=None if parents is None else ints(parents))
    cu, slots, positions, masks, info, after = step_ref.plan(lengths, new, parents, table, free, bs, N)
    assert got.cu.tolist() == cu
    assert got.info.tolist() == info
    assert got.slots.tolist() == slots
    assert got.positions.tolist() == positions
    if parents is None:
        assert got.masks is None
    else:
        assert got.masks.tolist() == masks
    assert np.array_equal(wide[:, :cols].cpu().numpy(), after)
    assert bool((wide[:, cols:] == -77).all())


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("lengths, new", [
    ([0], [1]), ([15], [1]), ([16], [1]), ([17], [30]), ([0, 5, 16, 31], [16, 0, 1, 64]),
    ([3] * 40, [5] * 40), ([100, 0, 47], [0, 0, 0])])
@pytest.mark.parametrize("bs", [16, 64])
def test_plan(tree, lengths, new, bs):
    N = sum(new)
    parents = random_parents(np.random.default_rng(1), new, N) if tree else None
    run_plan(lengths, new, parents, 12, bs, N, 200)


@pytest.mark.parametrize("tree", [False, True])
def test_plan_many_requests(tree):
    rng = np.random.default_rng(2)
    new = rng.integers(0, 65 if tree else 90, 777).tolist()
    lengths = rng.integers(0, 500, 777).tolist()
    N = sum(new)
    run_plan(lengths, new, random_parents(rng, new, N) if tree else None, 20, 32, N, 9000, seed=3, stride=23)


def test_plan_long_prompts_and_most_requests():
    run_plan([7, 0, 900], [5000, 1, 3001], None, 400, 16, 8002, 600, seed=4)
    B = 8192
    run_plan([1] * B, [1] * B, None, 2, 16, B, 1, seed=5)
    run_plan([16] * B, [2] * B, [-1, 0] * B, 2, 16, 2 * B, B, seed=6)


@pytest.mark.parametrize("tree", [False, True])
def test_plan_padding_shortage_and_bad_values(tree):
    def p(new, N):
        return random_parents(np.random.default_rng(7), new, N) if tree else None
    run_plan([5, 9], [3, 4], p([3, 4], 16), 3, 16, 16, 4)           # nine rows of padding
    run_plan([5, 9], [30, 40], p([30, 40], 50), 8, 16, 50, 20)      # fewer rows than tokens
    run_plan([14, 14, 14], [20, 20, 20], p([20] * 3, 60), 9, 16, 60, 3)  # free blocks run out
    run_plan([14, 3], [20, 60], p([20, 60], 80), 2, 16, 80, 9)      # columns run out
    run_plan([40, 3], [4, 4], p([4, 4], 8), 2, 16, 8, 9)            # a length beyond the table
    run_plan([-4, 3], [5, -2], p([5], 5), 2, 16, 5, 9)              # negative: zero
    run_plan([2, 0], [0, 0], p([], 6), 2, 16, 6, 0)                 # only padding, nothing free


def test_plan_parents_that_are_none():
    # itself, a later token, far out of range, below -1
    run_plan([4], [8], [-1, 1, 5, 99, -9, 3, 2 ** 31 - 1, -2 ** 31], 3, 16, 8, 4)
    chain = [-1] + list(range(63))
    run_plan([4, 4], [64, 70], chain + chain + [63] * 6, 9, 16, 134, 20)


def test_plan_repeats_itself():
    lengths, new, free = ints([5, 30]), ints([20, 9]), ints(range(50, 60))
    table = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    a = step.plan_step(lengths, new, table, free, 16, 29)
    first = table.clone()
    b = step.plan_step(lengths, new, table, free, 16, 29)
    assert torch.equal(first, table) and all(torch.equal(x, y) for x, y in zip(a, b) if x is not None)


# ---------------------------------------------------------------- norm and rotation

def run_rope(N, hq, hkv, D, rot, *, cache=torch.float16, bs=16, bias=False, norm=False, inter=False, pad=0,
             by_head=True, seed=0, positions=None, slots=None, rows=50, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    width = (hq + 2 * hkv) * D
    x = (scale * torch.randn((N, width + pad), generator=g)).cuda()[:, :width]
    nb = -(-N // bs) + 2
    ks, vs = step.paged_cache(nb, bs, hkv, D, cache)
    if not by_head:
        ks, vs = ks.contiguous(), vs.contiguous()
    ks.fill_(7.0), vs.fill_(9.0)
    positions = torch.randint(0, rows, (N,), generator=g).tolist() if positions is None else positions
    slots = torch.randperm(nb * bs, generator=g)[:N].tolist() if slots is None else slots
    t = step.rope_table(rows, rot)
    b = torch.randn(width, generator=g).cuda() if bias else None
    qw, kw = ((1 + torch.randn(D, generator=g)).cuda() for _ in range(2)) if norm else (None, None)
    q = step.qk_norm_rope(x, ints(positions), ints(slots), t, ks, vs, bias=b, q_weight=qw, k_weight=kw,
                          eps=1e-5, interleaved=inter)

    def np_(v):
        return None if v is None else v.cpu().numpy()
    h = step_ref.norm_rope(np_(x), hq, hkv, D, rot, inter, np_(b), np_(qw), np_(kw), 1e-5, positions, np_(t))
    # an element is a norm's factor (D / 8 + 8 roundings) times a sum of two
    # products (3): held against the pair's length, of at most the head's
    length = np.sqrt((h ** 2).sum(-1, keepdims=True))
    tol = (D / 8 + 16) * U * length + 1e-37
    got = q.double().cpu().numpy()
    assert got.shape == (N, hq, D)
    bad = np.isnan(h[:, :hq]) != np.isnan(got)
    assert not bad.any()
    assert (np.nan_to_num(np.abs(got - h[:, :hq])) <= np.nan_to_num(tol[:, :hq])).all()
    half = 2.0 ** -11 if cache == torch.float16 else 2.0 ** -8
    tiny = 2.0 ** -25 if cache == torch.float16 else 1e-38
    for c, lo, fill in ((ks, hq, 7.0), (vs, hq + hkv, 9.0)):
        want = np.full((nb * bs, hkv, D), fill)
        room = np.zeros((nb * bs, hkv, 1))
        for n, s in enumerate(slots):
            if 0 <= s < nb * bs:
                want[s] = h[n, lo:lo + hkv]
                room[s] = tol[n, lo:lo + hkv]
        got = c.reshape(nb * bs, hkv, D).double().cpu().numpy()
        assert (np.isnan(got) == np.isnan(want)).all()
        err = np.nan_to_num(np.abs(got - want))
        assert (err <= np.nan_to_num(room * 1.01 + half * np.abs(want)) + tiny).all(), float(err.max())


@pytest.mark.parametrize("D, rot", [(8, 8), (64, 64), (64, 32), (80, 80), (96, 96), (96, 48), (128, 128), (128, 64),
                                    (128, 0), (256, 256), (256, 64), (512, 512)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
def test_rope(D, rot, inter, cache):
    for i, (bias, norm) in enumerate(((False, False), (True, False), (False, True), (True, True))):
        run_rope(5, 6, 2, D, rot, inter=inter, cache=cache, bias=bias, norm=norm, seed=i)


@pytest.mark.parametrize("N", [1, 2, 7, 64, 333])
@pytest.mark.parametrize("hq, hkv", [(1, 1), (7, 1), (32, 4), (28, 4), (12, 12)])
def test_rope_sizes(N, hq, hkv):
    run_rope(N, hq, hkv, 64, 64, norm=True, seed=N, bs=32)
    run_rope(N, hq, hkv, 128, 128, norm=N % 2 == 0, bias=True, cache=torch.bfloat16, seed=N)


def test_rope_strides_layouts_and_missing_slots():
    for by_head in (False, True):
        for pad in (1, 4, 640):
            run_rope(9, 4, 2, 64, 64, pad=pad, by_head=by_head, norm=True)
    run_rope(6, 4, 2, 128, 128, slots=[-1, 3, -5, 10 ** 9, 17, 2 ** 31 - 1], norm=True)
    run_rope(6, 4, 2, 128, 128, positions=[0, -1, 49, 50, 2 ** 31 - 1, -2 ** 31], norm=True)
    run_rope(4, 4, 2, 64, 64, scale=1e-30, norm=True)  # far below eps
    run_rope(4, 4, 2, 64, 64, scale=1e-6)              # subnormal in fp16


def test_rope_values_beyond_fp16_are_infinite():
    x = torch.full((1, 3 * 64), 1e5, device="cuda")
    k, v = step.paged_cache(1, 16, 1, 64)
    step.qk_norm_rope(x, ints([0]), ints([0]), step.rope_table(1, 64), k, v)
    assert bool(torch.isinf(v[0, 0]).all()) and not v[0, 1:].any()


# ---------------------------------------------------------------- tree attention

def tree_masks(rng, new):
    out = []
    for n in new:
        m = []
        for i in range(n):
            p = int(rng.integers(-1, i)) if i else -1
            m.append((1 << i) | (m[p] if p >= 0 else 0))
        out += [v - (1 << 64) if v >> 63 else v for v in m]
    return out


class Case:
    """Requests over a cache whose every other value is NaN."""

    def __init__(self, lengths, new, hq, hkv, D, *, cache=torch.float16, bs=16, tree=False, seed=0, pad=0,
                 by_head=True, spread=2.0, extra_cols=2, padding=0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.new = lengths, new
        self.cu = [0] + np.cumsum(new).tolist()
        self.N = self.cu[-1] + padding
        cols = max(1, max(-(-(a + b) // bs) for a, b in zip(lengths, new))) + extra_cols
        need = [-(-(a + b) // bs) for a, b in zip(lengths, new)]
        nb = sum(need) + 3
        ids = rng.permutation(nb)
        self.table = torch.full((len(new), cols), 2 ** 30, dtype=torch.int32)  # never to be followed
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = torch.from_numpy(ids[at:at + n].astype(np.int32))
            at += n
        self.k, self.v = (c.fill_(math.nan) for c in step.paged_cache(nb, bs, hkv, D, cache, device="cpu"))
        for b, n in enumerate(need):
            for t in range(lengths[b] + new[b]):
                p = int(self.table[b, t // bs])
                self.k[p, t % bs] = torch.randn((hkv, D), generator=g)
                self.v[p, t % bs] = torch.randn((hkv, D), generator=g)
        if not by_head:
            self.k, self.v = self.k.contiguous(), self.v.contiguous()
        self.q = spread * torch.randn((self.N, hq, D + 0), generator=g)
        self.pad, self.masks, self.D, self.by_head = pad, None, D, by_head
        if tree:
            self.masks = torch.tensor(tree_masks(rng, new) + [-1] * padding, dtype=torch.int64)

    def cuda_cache(self):
        return tuple(c.transpose(1, 2).contiguous().cuda().transpose(1, 2) if self.by_head else c.cuda()
                     for c in (self.k, self.v))

    def run(self, **kw):
        k, v = self.cuda_cache()
        q = self.q.cuda()
        if self.pad:  # tokens further apart than their heads
            wide = torch.full((self.N, q[0].numel() + self.pad), math.nan, device="cuda")
            wide[:, :q[0].numel()] = q.flatten(1)
            q = wide[:, :q[0].numel()].view(self.N, *q.shape[1:]) if self.N == 1 else \
                wide.as_strided(q.shape, (wide.stride(0), self.D, 1))
        return step.tree_attention(q, k, v, self.table.cuda(), ints(self.lengths), ints(self.cu),
                                   None if self.masks is None else self.masks.cuda(), **kw)

    def check(self, **kw):
        out = self.run(**kw).double().cpu()
        scale = kw.get("scale", self.D ** -0.5)
        want = step_ref.attention(self.q, self.k, self.v, self.table, self.lengths, self.cu,
                                  None if self.masks is None else self.masks.tolist(), scale)
        # a score is a sum of D products of a query of 22 bits and more in fp32:
        # off by at most 2^-20 of sum |q k|; a probability by twice that (its own
        # and the sum's) and the exponential's, the parts' and the keys' sums' roundings
        fine = torch.nan_to_num(self.k.float(), 0.0, 0.0, 0.0)
        kmax = float(fine.norm(dim=-1).max())
        ds = 2.0 ** -20 * abs(scale) * float(self.q.norm(dim=-1).max()) * kmax
        most = max(a + b for a, b in zip(self.lengths, self.new))
        vmax = float(torch.nan_to_num(self.v.float(), 0.0, 0.0, 0.0).abs().max())
        tol = vmax * (2 * ds + (32 + most / 16) * U)
        assert bool((torch.isnan(out) == torch.isnan(want)).all())
        err = float(torch.nan_to_num(out - want, 0.0, 0.0, 0.0).abs().max()) if out.numel() else 0.0
        assert err <= tol, (err, tol)
        return out


HEADS = [(1, 1), (4, 1), (7, 1), (8, 2), (6, 6), (28, 4)]


@pytest.mark.parametrize("D", [64, 96, 128, 256])
@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq, hkv", HEADS)
def test_attention_heads(D, cache, hq, hkv):
    Case([37], [1], hq, hkv, D, cache=cache).check()
    Case([0, 130, 5], [3, 9, 6], hq, hkv, D, cache=cache, tree=True, seed=1).check()


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 300, 1025])
@pytest.mark.parametrize("new", [1, 2, 5, 17])
def test_attention_lengths(length, new):
    Case([length], [new], 8, 2, 64, seed=length).check(max_new=new)
    Case([length, 3, length], [new, 1, new], 4, 2, 128, cache=torch.bfloat16, bs=32, tree=True,
         seed=length).check(max_new=new)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 3, 4, 7, 8, 9, 16, 33, 63, 64])
def test_attention_trees(D, cache, new):
    Case([200, 77], [new, max(1, new // 2)], 8, 2, D, cache=cache, tree=True, seed=new).check(max_new=new)
    Case([90], [new], 7, 1, D, cache=cache, tree=False, seed=new).check(max_new=new)


@pytest.mark.parametrize("bs", [16, 32, 64, 256, 1024])
def test_attention_block_sizes_layouts_and_strides(bs):
    for by_head in (True, False):
        Case([70, 1100], [5, 2], 8, 4, 64, bs=bs, by_head=by_head, tree=True, pad=12).check()
        Case([70, 33], [5, 2], 8, 4, 128, bs=bs, by_head=by_head, pad=1, cache=torch.bfloat16).check()


def test_attention_ragged_batches():
    rng = np.random.default_rng(5)
    for seed in range(6):
        B = int(rng.integers(2, 40))
        lengths = [int(v) for v in np.where(rng.random(B) < 0.2, 0, rng.integers(0, 400, B))]
        new = [int(v) for v in rng.integers(0, 12, B)]
        if sum(new) == 0:
            new[0] = 1
        out = Case(lengths, new, 6, 2, 64, tree=seed % 2 == 0, seed=seed, padding=seed).check()
        assert not out[sum(new):].any() or seed == 0


def test_attention_many_requests():
    # more requests than work-groups' lanes
    rng = np.random.default_rng(6)
    B = 700
    Case(rng.integers(0, 40, B).tolist(), rng.integers(0, 3, B).tolist(), 2, 1, 64, seed=7).check(max_new=2)


def test_attention_long_context_in_many_parts():
    Case([30011], [3], 4, 1, 64, bs=64, tree=True, seed=8).check(max_new=3)
    Case([9000, 100, 20000], [2, 7, 1], 4, 2, 128, bs=32, cache=torch.bfloat16, seed=9).check()


def test_attention_more_than_64_tokens_of_a_chain():
    Case([50, 0], [70, 131], 4, 2, 64, seed=10).check()
    # with masks, tokens from the 65th on are seen by none
    c = Case([50], [70], 4, 2, 64, seed=10, tree=False)
    c.masks = torch.tensor([(1 << min(i, 63)) - 1 for i in range(70)], dtype=torch.int64)
    c.check()


def test_attention_max_new_is_only_a_hint():
    c = Case([100, 20], [21, 4], 8, 2, 64, tree=True, seed=11)
    for hint in (0, 1, 4, 21, 64, 10 ** 6):
        c.check(max_new=hint)


def test_attention_rows_that_see_nothing_are_zero():
    c = Case([0, 0, 40], [4, 1, 3], 8, 2, 64, tree=True, seed=12)
    c.masks[:] = 0
    out = c.check()
    assert not out[:5].any() and out[5:].abs().sum() > 0
    c.masks[1] = 1  # one of a tile's rows sees a key
    out = c.check()
    assert not out[0].any() and bool(out[1].any())


@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("length", [0, 30, 140])
def test_attention_masked_values_take_no_part(cache, what, length):
    # token 2's key and value are not finite: only the tokens that see it feel it
    c = Case([length], [6], 8, 2, 64, cache=cache, tree=True, seed=13)
    c.masks = torch.tensor([1, 3, 7, 9, 0b10011, 0b100111], dtype=torch.int64)
    p, r = int(c.table[0, (length + 2) // 16]), (length + 2) % 16
    c.v[p, r, :, 5] = what
    out = c.check()
    assert bool(torch.isfinite(out[[0, 1, 3, 4]]).all())
    assert not torch.isfinite(out[[2, 5], :, 5]).any() and bool(torch.isfinite(out[[2, 5], :, 6:]).all())
    c.v[p, r, :, 5] = 0.5
    c.k[p, r] = what
    out = c.run().cpu()
    assert bool(torch.isfinite(out[[0, 1, 3, 4]]).all())


def test_attention_non_finite_cached_values_reach_every_row():
    c = Case([40], [3], 4, 2, 64, seed=14)
    p = int(c.table[0, 0])
    c.v[p, 3, 0, 7] = math.inf
    c.v[p, 4, 1, 9] = math.nan
    c.check()


@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
def test_attention_scores_far_apart(cache):
    # one key's score lies far above the others', first, last and in between
    for at in (0, 35, 199, 203):
        c = Case([200], [4], 4, 1, 64, cache=cache, seed=15)
        p = int(c.table[0, at // 16])
        c.k[p, at % 16] = 40.0 * torch.sign(c.q[3, 0])
        c.check()
    Case([300], [4], 4, 2, 128, cache=cache, seed=16, spread=1e-20).check()
    Case([300], [4], 4, 2, 128, cache=cache, seed=17).check(scale=-0.3)
    Case([300], [4], 4, 2, 128, cache=cache, seed=17).check(scale=0.0)


def test_attention_of_fp16_extremes():
    c = Case([100], [3], 4, 2, 64, seed=18, spread=1e-3)
    c.v[torch.isfinite(c.v)] = 65504.0
    out = c.check()
    assert bool((out - 65504.0).abs().max() <= 65504.0 * 40 * U)
    c = Case([100], [3], 4, 2, 64, seed=18)
    fine = torch.isfinite(c.v)
    c.v[fine] = c.v[fine] * 2.0 ** -20  # subnormal
    c.check()
    c = Case([100], [3], 4, 2, 64, seed=18, spread=1e30)  # a query's bits lie in its exponent too
    fine = torch.isfinite(c.k)
    c.k[fine] = c.k[fine] * 2.0 ** -14
    c.check(scale=1e-27)


def test_attention_of_a_long_cache_past_32_bit_offsets():
    # 5 GiB of keys; the request's blocks lie at the end
    nb, bs, hkv, D = 41000, 64, 8, 128
    k = torch.empty((nb, hkv, bs, D), dtype=torch.float16, device="cuda").transpose(1, 2)
    v = torch.empty((nb, hkv, bs, D), dtype=torch.float16, device="cuda").transpose(1, 2)
    k[:3], v[:3] = 5.0, 5.0
    k[-3:], v[-3:] = torch.randn_like(k[-3:]), torch.randn_like(v[-3:])
    table = ints([[nb - 2, nb - 1, nb - 3]])
    q = 2 * torch.randn((2, 16, D), device="cuda")
    x = torch.randn((2, (16 + 2 * hkv) * D), device="cuda")
    plan = step.plan_step(ints([150]), ints([2]), table, ints([0]), bs, 2)
    assert plan.slots.tolist() == [(nb - 3) * 64 + 22, (nb - 3) * 64 + 23]
    q = step.qk_norm_rope(x, plan.positions, plan.slots, step.rope_table(160, D), k, v)
    out = step.tree_attention(q, k, v, table, ints([150]), plan.cu)
    want = step_ref.attention(q, k[-3:].cpu(), v[-3:].cpu(), torch.tensor([[1, 2, 0]]), [150], [0, 2], None, D ** -0.5)
    assert float((out.cpu().double() - want).abs().max()) < 1e-4


def test_attention_repeats_to_the_bit():
    c = Case([5000, 333, 0], [9, 20, 4], 8, 2, 128, tree=True, seed=19, bs=32)
    a = c.run()
    for _ in range(3):
        assert torch.equal(a, c.run())


# ---------------------------------------------------------------- log probabilities

def run_logprobs(x, targets, top):
    got = step.token_logprobs(x, ints(targets), top=top)
    t = np.array(targets)
    lp, H, tokens, tl = step_ref.logprobs(x, t, top)
    V = x.shape[1]
    # (x - m) - log s: the sum's V / 256 additions a lane and 24 to join them, an
    # exponential's 2 + |x - m| and the last differences' roundings
    f = torch.nan_to_num(x.float(), 0.0, 0.0, 0.0).clamp(-1e4, 1e4)
    spread = float(f.max() - f.min())

    def near(a, b, what):
        a = a.double().cpu().numpy()
        assert (np.isnan(a) == np.isnan(b)).all(), what
        inf = np.isinf(b)
        assert (a[inf] == b[inf]).all(), what
        ok = ~(np.isnan(b) | inf)
        room = (V / 256 + 40 + 4 * min(spread, 90.0)) * U * np.maximum(1.0, np.log(V)) + 4 * U * np.abs(b[ok])
        assert (np.abs(a[ok] - b[ok]) <= room).all(), (what, float(np.abs(a[ok] - b[ok]).max()))

    near(got.logprobs, lp, "logprobs")
    near(got.entropy, H, "entropy")
    if top:
        assert np.array_equal(got.top_tokens.cpu().numpy(), tokens)
        near(got.top_logprobs, tl, "top")
    else:
        assert got.top_tokens is None and got.top_logprobs is None


@pytest.mark.parametrize("V", [1, 2, 63, 255, 256, 4095, 4096, 4097, 8193, 50257, 152064])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_logprobs(V, dtype):
    g = torch.Generator().manual_seed(V)
    for M, top in ((1, min(V, 5)), (3, min(V, 64)), (2, 0)):
        x = (3 * torch.randn((M, V), generator=g)).to(dtype).cuda()
        run_logprobs(x, torch.randint(0, V, (M, 2), generator=g).tolist(), top)


def test_logprobs_many_rows_and_strides():
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((1500, 1003), generator=g).cuda()
    run_logprobs(wide[:, :1000], [[m % 1000] for m in range(1500)], 7)
    run_logprobs(wide[3:40, 1:998], [5] * 37, 20)
    half = wide.half()
    run_logprobs(half[:, 3:1000], [m % 997 for m in range(1500)], 3)
    run_logprobs(half[:700:7], [[0, 1002, 5]] * 100, 64)


def test_logprobs_ties_go_to_the_lowest_token():
    for V in (300, 5000, 40000):
        x = torch.zeros((2, V), device="cuda")
        x[1, ::3] = 1.0
        run_logprobs(x, [0, V - 1], 64)
        x[0, ::2] = -0.0  # equal to 0
        run_logprobs(x, [0, 1], 64)
        run_logprobs(x.half(), [0, 1], 64)
    up = torch.arange(9000.0, device="cuda")[None] / 1000
    run_logprobs(torch.cat([up, up.flip(1)]), [8999, 0], 64)


def test_logprobs_masked_rows():
    inf = math.inf
    g = torch.Generator().manual_seed(2)
    for V in (100, 9000, 50000):
        x = torch.randn((6, V), generator=g).cuda()
        x[0] = -inf                      # nothing is left
        x[1, 1:] = -inf                  # one token is left
        x[2, torch.arange(V).cuda() % 50 != 7] = -inf  # two are (and more)
        x[3] = -3.402823466e38           # the type's lowest value
        x[3, 5] = 1.0
        x[4] = -3.402823466e38
        x[5, :V // 2] = -inf
        run_logprobs(x, [[0, 1]] * 6, 10)
        x[0, V // 2] = math.nan
        x[1, 7] = inf
        x[2, 3] = -math.nan
        x[2, 50] = math.nan
        run_logprobs(x, [[0, 7]] * 6, 10)


def test_logprobs_where_every_part_of_a_row_has_all_the_largest():
    # the largest logits lie in the last token's neighbourhood, then spread evenly
    g = torch.Generator().manual_seed(3)
    for V, M in ((40000, 2), (40000, 300), (70000, 600)):
        x = torch.randn((M, V), generator=g).cuda()
        x[:, -64:] += 20
        run_logprobs(x, [V - 1] * M, 64)
        x[:, ::V // 2000] += 40
        run_logprobs(x, [0] * M, 64)
    steps = torch.arange(120000.0, device="cuda")  # rising by units: every chunk has larger ones
    run_logprobs(steps[None].repeat(3, 1) / 1024, [0, 1, 119999], 64)


def test_logprobs_targets_outside_the_vocabulary():
    x = torch.randn((2, 777), device="cuda")
    run_logprobs(x, [[0, -1, 776], [777, 2 ** 31 - 1, -2 ** 31]], 3)


def test_logprobs_without_targets():
    x = torch.randn((4, 300), device="cuda")
    r = step.token_logprobs(x, top=2)
    assert r.logprobs is None and torch.equal(r.top_tokens[:, 0].long(), x.argmax(1))
    with pytest.raises(RuntimeError, match="at most 64"):
        step.token_logprobs(x, top=65)


# ---------------------------------------------------------------- together

def step_of(state):
    lengths, new, table, free, parents, x, t, k, v, logits, targets = state
    N = x.shape[0]
    plan = step.plan_step(lengths, new, table, free, 16, N, parents=parents)
    q = step.qk_norm_rope(x, plan.positions, plan.slots, t, k, v)
    o = step.tree_attention(q, k, v, table, lengths, plan.cu, plan.masks, max_new=9)
    r = step.token_logprobs(logits, targets, top=4)
    return o, r.logprobs, r.entropy, r.top_logprobs, r.top_tokens


def state_of(seed):
    g = torch.Generator().manual_seed(seed)
    hq, hkv, D, bs = 8, 2, 64, 16
    lengths, new = [700, 0, 33], [9, 4, 1]
    N = sum(new)
    table = torch.zeros((3, 50), dtype=torch.int32)
    table[0, :44] = torch.arange(44)
    table[2, :3] = torch.arange(44, 47)
    parents = random_parents(np.random.default_rng(seed), new, N)
    k, v = step.paged_cache(60, bs, hkv, D)
    k[:47] = torch.randn((47, bs, hkv, D), generator=g).cuda().half()
    v[:47] = torch.randn((47, bs, hkv, D), generator=g).cuda().half()
    return (ints(lengths), ints(new), table.cuda(), ints(range(47, 60)), ints(parents),
            torch.randn((N, (hq + 2 * hkv) * D), generator=g).cuda(), step.rope_table(800, D), k, v,
            torch.randn((N, 32000), generator=g).cuda(), ints([i * 7 for i in range(N)]))


def test_step_on_another_stream_and_in_a_graph():
    state = state_of(1)
    want = [t.clone() for t in step_of(state)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step_of(state)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.cuda.stream(side):
        step.reserve()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        kept = step_of(state)
    for r in range(4):
        other = state_of(2 + r)  # new inputs in the same buffers
        for a, b in zip(state, other):
            a.copy_(b)
        fresh = step_of(other)  # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(fresh, kept):
            assert torch.equal(a, b), r


def test_capture_without_a_workspace_is_refused():
    from forge_amd import _lib
    state = state_of(3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert _lib.lib().fq_release_workspace(side.cuda_stream) == 0  # (streams are reused)
    q, cu = state[5].view(14, 12, 64)[:, :8].contiguous(), ints([0, 9, 13, 14])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(_lib.FqError, match="workspace"):
            step.tree_attention(q, state[7], state[8], state[2], state[0], cu)


def test_python_refusals():
    s = state_of(4)
    lengths, new, table, free, parents, x, t, k, v, logits, targets = s
    q = torch.zeros((14, 8, 64), device="cuda")
    cu = ints([0, 9, 13, 14])
    for bad, match in (
            (lambda: step.plan_step(lengths.long(), new, table, free, 16, 14), "lengths"),
            (lambda: step.plan_step(lengths, new[:2], table, free, 16, 14), "new_tokens"),
            (lambda: step.plan_step(lengths, new, table[:2], free, 16, 14), "block_table"),
            (lambda: step.plan_step(lengths, new, table.t(), free, 16, 14), "block_table"),
            (lambda: step.plan_step(lengths, new, table, free, 16, 14, parents=parents[:3]), "parents"),
            (lambda: step.plan_step(lengths, new, table, free, 15, 14), "invalid shape"),
            (lambda: step.qk_norm_rope(x.half(), cu, cu, t, k, v), "fp32"),
            (lambda: step.qk_norm_rope(x[:, :-64], cu, cu, t, k, v), "do not hold"),
            (lambda: step.qk_norm_rope(x, targets[:3], targets, t, k, v), "positions"),
            (lambda: step.qk_norm_rope(x, targets, targets, t, k, v.contiguous()), "alike"),
            (lambda: step.qk_norm_rope(x, targets, targets, t, k.float(), v.float()), "fp16 or bf16"),
            (lambda: step.qk_norm_rope(x, targets, targets, t, k, v, bias=x[0, :-1]), "bias"),
            (lambda: step.tree_attention(q.half(), k, v, table, lengths, cu), "fp32"),
            (lambda: step.tree_attention(q[:, :7], k, v, table, lengths, cu), "do not share"),
            (lambda: step.tree_attention(q, k, v, table, lengths, cu[:3]), "cu"),
            (lambda: step.tree_attention(q, k, v, table, lengths, cu, masks=targets), "masks"),
            (lambda: step.tree_attention(q.transpose(0, 1), k, v, table, lengths, cu), "contiguous"),
            (lambda: step.token_logprobs(logits, targets.long()), "targets"),
            (lambda: step.token_logprobs(logits.t()), "contiguous rows")):
        with pytest.raises(RuntimeError, match=match):
            bad()
