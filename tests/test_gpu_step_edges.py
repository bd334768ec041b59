"""Step operators at the edges of what device memory may hold: block tables with
entries that are no block, lengths beyond a table, keys that are infinite."""
from __future__ import annotations

import math

import pytest
import torch

from forge_amd import step
from test_gpu_step import U, Case, ints

pytestmark = pytest.mark.gpu

NONE = [-1, -2 ** 31, 2 ** 31 - 1, 2 ** 30]  # (and the number of blocks) are no blocks


def plain(c, scale=None):
    """fp64 [N, hq, D]: token by token over the keys that it sees and that lie in a block;
    a key that scores -inf has no weight, and where none has any the row is zeros."""
    scale = c.D ** -0.5 if scale is None else scale
    nb, bs, hkv = c.k.shape[:3]
    hq = c.q.shape[1]
    out = torch.zeros((c.N, hq, c.D), dtype=torch.float64)
    for b, ln in enumerate(c.lengths):
        t0, n = c.cu[b], c.cu[b + 1] - c.cu[b]
        keys = min(ln + n, c.table.shape[1] * bs)
        pages = c.table[b, :-(-keys // bs)].long()
        fine = (pages >= 0) & (pages < nb)
        there = fine.repeat_interleave(bs)[:keys]
        k, v = (x[torch.where(fine, pages, 0)].flatten(0, 1)[:keys].double() for x in (c.k, c.v))
        j = torch.arange(keys) - ln  # a key's number among the new tokens
        for i in range(n):
            if c.masks is None:
                see = j <= i
            else:
                m = int(c.masks[t0 + i])
                see = (j < 0) | torch.tensor([0 <= x < 64 and m >> x & 1 == 1 for x in j.tolist()], dtype=torch.bool)
            see = see & there
            if not see.any():
                continue
            kk, vv = (x[see].repeat_interleave(hq // hkv, 1) for x in (k, v))
            s = (c.q[t0 + i].double()[None] * kk).sum(-1) * scale
            top = s.amax(0)
            w = torch.where(s == -math.inf, torch.zeros_like(s), torch.exp(s - top))
            total = w.sum(0)
            o = (w[..., None] * vv).sum(0) / torch.where(total == 0, 1.0, total)[:, None]
            out[t0 + i] = torch.where(torch.isnan(s).any(0) | (top == math.inf), math.nan, o.T).T
    return out


def near(c, out, want, scale=None):
    # as Case.check: scores off by at most 2^-20 of |q| |k|, probabilities by twice
    # that and the roundings of the exponential, of the parts and of the keys' sums
    def fine(x):
        return torch.nan_to_num(x.float(), 0.0, 0.0, 0.0)
    ds = 2.0 ** -20 * (scale or c.D ** -0.5) * float(c.q.norm(dim=-1).max()) * float(fine(c.k).norm(dim=-1).max())
    most = max(a + b for a, b in zip(c.lengths, c.new))
    tol = float(fine(c.v).abs().max()) * (2 * ds + (32 + most / 16) * U)
    out = out.double().cpu()
    assert bool((torch.isnan(out) == torch.isnan(want)).all())
    err = float(torch.nan_to_num(out - want, 0.0, 0.0, 0.0).abs().max())
    assert err <= tol, (err, tol)


# (up to 16, 32 and 64 rows to a tile; whole and cut items)
SHAPES = [(64, 2, 1), (64, 2, 5), (64, 2, 20), (128, 2, 3), (128, 2, 7), (128, 2, 24), (96, 1, 9), (256, 2, 3), (256, 2, 11)]


@pytest.mark.parametrize("D, hkv, new", SHAPES)
@pytest.mark.parametrize("cache, tree", [(torch.float16, True), (torch.bfloat16, False)])
@pytest.mark.parametrize("what", [5.0, math.nan])
def test_keys_without_a_block_are_not_seen(D, hkv, new, cache, tree, what):
    for lengths, bs, holes in (([70, 33], 16, [(0, 1), (1, 0)]),           # one in the context, one the first
                               ([160, 9], 32, [(0, 0), (0, 3), (0, 5)]),   # the last: the new tokens'
                               ([3000, 700], 16, [(0, 0), (0, 100), (0, 101), (0, 150), (1, 43)]),
                               ([130, 0], 16, [(1, x) for x in range(2)])):
        c = Case(lengths, [new, max(1, new - 2)], 4 * hkv, hkv, D, cache=cache, bs=bs, tree=tree, seed=new)
        nb = c.k.shape[0]
        free = [int(c.table[b, x]) for b, x in holes]
        for i, (b, x) in enumerate(holes):
            c.table[b, x] = (NONE + [nb])[i % 5]
        # what a clamp to the cache would read (blocks of nobody, or of the other request)
        for p in (0, nb - 1):
            if p in free or p not in c.table:
                c.k[p], c.v[p] = what, what
        near(c, c.run(max_new=new), plain(c))


def test_a_request_whose_every_block_is_missing_gets_zeros():
    c = Case([40, 50], [3, 2], 8, 2, 64, seed=2)
    c.table[0] = -1
    out = c.run()
    assert not out[:3].any() and bool(out[3:].any())
    near(c, out, plain(c))


def test_tokens_that_found_no_block_take_no_part():
    # the free blocks run out within the second request: its further tokens have no
    # slot, and the first block, another request's, stays out of their attention
    bs, hkv, hq, D, lengths, new = 16, 2, 8, 64, [16, 14], [4, 20]
    g = torch.Generator().manual_seed(3)
    k, v = step.paged_cache(4, bs, hkv, D)
    k[:3], v[:3] = (torch.randn((3, bs, hkv, D), generator=g).cuda().half() for _ in range(2))
    table = ints([[0, 9, 9], [2, 9, 9]])
    plan = step.plan_step(ints(lengths), ints(new), table, ints([1]), bs, 24)
    assert plan.info.tolist() == [1, 2] and table.tolist() == [[0, 1, 9], [2, -1, -1]]
    assert plan.slots.tolist() == [16, 17, 18, 19] + [46, 47] + [-1] * 18
    x = torch.randn((24, (hq + 2 * hkv) * D), generator=g).cuda()
    q = step.qk_norm_rope(x, plan.positions, plan.slots, step.rope_table(64, D), k, v)
    c = Case(lengths, new, hq, hkv, D)
    c.q, c.k, c.v, c.table = q.cpu(), k.cpu(), v.cpu(), table.cpu()
    near(c, step.tree_attention(q, k, v, table, ints(lengths), plan.cu), plain(c))


@pytest.mark.parametrize("D, hkv, new", SHAPES)
@pytest.mark.parametrize("tree", [False, True])
def test_lengths_beyond_the_table_end_with_it(D, hkv, new, tree):
    for cols, bs, lengths in ((3, 16, [200, 20]), (5, 16, [81, 10 ** 6]), (1, 16, [2 ** 31 - 1, 17]), (67, 16, [1071, 5000]),
                              (3, 64, [191, 300])):
        c = Case([min(n, cols * bs - 64) if cols * bs > 64 else 0 for n in lengths], [new, 2], 4 * hkv, hkv, D, bs=bs, tree=tree, seed=new)
        g = torch.Generator().manual_seed(new)
        nb = 2 * cols + 1
        c.k, c.v = (torch.randn((nb, hkv, bs, D), generator=g).to(c.k.dtype).transpose(1, 2) for _ in range(2))
        c.table = torch.randperm(nb, generator=g)[:2 * cols].view(2, cols).int()
        c.lengths = lengths
        out, want = c.run(max_new=new), plain(c)
        c.lengths = [cols * bs - n for n in c.new]  # (the keys that there are)
        near(c, out, want)


@pytest.mark.parametrize("D, hkv, new", SHAPES)
@pytest.mark.parametrize("cache", [torch.float16, torch.bfloat16])
def test_infinite_keys_score_as_they_do(D, hkv, new, cache):
    # a key with an infinite element scores -inf, and has no weight, or +inf, whose
    # softmax is NaN, by the sign of the query's element
    for lengths in ([40, 3], [2000, 0]):
        for at in (0, 17, lengths[0] - 1, lengths[0]):
            c = Case(lengths, [new, 2], 4 * hkv, hkv, D, cache=cache, tree=True, seed=new)
            p = int(c.table[0, at // 16])
            c.k[p, at % 16, 0, 5] = math.inf
            c.q[:, 0, 5] = c.q[:, 0, 5].abs()
            c.q[:, 1, 5] = -c.q[:, 1, 5].abs()
            want = plain(c)
            assert bool(torch.isnan(want[:, 0]).any()) and bool(torch.isfinite(want[:, 1]).all())
            near(c, c.run(max_new=new), want)


def test_keys_that_all_score_minus_infinity_give_zeros():
    c = Case([37], [3], 4, 2, 64, seed=4)
    c.q = c.q.abs() + 0.1
    c.k[torch.isfinite(c.k)] = -math.inf
    assert not c.run().any()


def test_slots_past_the_largest_int_are_none():
    # (a block's number times the block's size does not fit: another block's slot)
    table = ints([[2 ** 27, 3], [2 ** 31 - 1, 2 ** 27 - 1]])
    plan = step.plan_step(ints([14, 3]), ints([4, 2]), table, ints([2 ** 28 + 1]), 16, 6)
    assert plan.slots.tolist() == [-1, -1, -1, -1, -1, -1]
    plan = step.plan_step(ints([14, 17]), ints([1, 2]), table, ints([]), 16, 3)
    assert plan.slots.tolist() == [-1, (2 ** 27 - 1) * 16 + 1, (2 ** 27 - 1) * 16 + 2]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_calls_go_to_the_tensors_device():
    from test_gpu_step import state_of, step_of
    want = step_of(state_of(5))
    there = [x.to("cuda:1") for x in state_of(5)]
    there[7], there[8] = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in there[7:9])
    assert torch.cuda.current_device() == 0
    got = step_of(there)
    assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    assert all(x.device.index == 1 and torch.equal(x.cpu(), y.cpu()) for x, y in zip(got, want))
