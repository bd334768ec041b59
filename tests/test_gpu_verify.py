"""verify_draft on the GPU against the plain 64-bit walk, its distribution, and the operators
of a sampled draft together: plan, norm and rotation into 8 bits, attention with a window,
verification, the accepted branch's move."""
from __future__ import annotations

import math
import os
import runpy

import numpy as np
import pytest
import torch

import step8_ref
from forge_amd import step

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def draft(new, V, *, tree, probs, seed, dtype=torch.float32, sharp=3.0, pad=0, padding=0, easy=0.6):
    """Logits, tokens, cu, uniforms, parents, draft probabilities: tokens likely under their parent's row."""
    rng = np.random.default_rng(seed)
    N = sum(new) + padding
    x = torch.from_numpy(sharp * rng.standard_normal((N, V + pad))).to(dtype)[:, :V]
    cu = [0] + np.cumsum(new).tolist()
    parents, tokens = [0] * N, [0] * N
    q = np.zeros((N, V))
    for t0, n in zip(cu, new):
        for i in range(n):
            up = (int(rng.integers(max(0, i - 4), i)) if tree else i - 1) if i else -1
            parents[t0 + i] = up
            row = x[t0 + max(up, 0)].double().numpy()
            d = np.exp(row - row.max()) * np.exp(0.7 * rng.standard_normal(V))
            q[t0 + i] = (d / d.sum()).astype(np.float32)
            tokens[t0 + i] = int(rng.choice(V, p=q[t0 + i].astype(np.float64) / q[t0 + i].astype(np.float64).sum())) \
                if rng.random() > easy or probs else int(row.argmax())
    u = rng.random(N).astype(np.float32)
    u[u == 1] = 0.5
    return x, tokens, cu, u, parents if tree else None, q if probs else None


def check(x, tokens, cu, u, parents, q, temperature=None):
    N, V = x.shape
    dx = x.cuda()
    if x.stride(0) != V and N > 1:  # rows further apart, what is between them NaN
        wide = torch.full((N, x.stride(0)), math.nan, dtype=x.dtype, device="cuda")
        wide[:, :V] = dx
        dx = wide[:, :V]
    qq = None
    if q is not None:
        qq = torch.from_numpy(q).float().cuda()
        q = qq.cpu().double().numpy()
    got = step.verify_draft(dx, ints(tokens), ints(cu), torch.from_numpy(u).cuda(),
                            parents=None if parents is None else ints(parents), draft_probs=qq,
                            temperature=None if temperature is None else torch.tensor(temperature, device="cuda"))
    temps = None if temperature is None else np.float32(temperature).astype(np.float64)
    accepted, path, following = step8_ref.verify(x.double().numpy(), tokens, cu, u.astype(np.float64), parents, q, temps)
    assert got.accepted.tolist() == accepted
    assert got.path.tolist() == path
    assert got.next_tokens.tolist() == following
    return got


KINDS = [(False, False), (False, True), (True, False)]


@pytest.mark.parametrize("tree, probs", KINDS)
@pytest.mark.parametrize("V", [1, 2, 17, 63, 1000, 4095, 4096, 4097, 12289, 32000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_sizes(tree, probs, V, dtype):
    for seed in range(3):
        check(*draft([6, 1, 9], V, tree=tree, probs=probs, seed=seed, dtype=dtype, pad=seed * 3, padding=seed))


@pytest.mark.parametrize("tree, probs", KINDS)
@pytest.mark.parametrize("new", [[1], [2], [64], [1] * 50, [0, 3, 0, 0, 7], [63, 5, 64]])
def test_requests(tree, probs, new):
    for seed in range(4):
        check(*draft(new, 300, tree=tree, probs=probs, seed=seed, easy=0.95))


@pytest.mark.parametrize("tree, probs", KINDS)
def test_temperatures(tree, probs):
    for seed in range(6):
        check(*draft([9, 5, 7, 1, 8], 500, tree=tree, probs=probs, seed=seed, easy=0.9),
              temperature=[0.0, 0.7, 1.9, 0.0, -3.0])


def test_many_requests():
    for probs in (False, True):
        check(*draft([1 + b % 3 for b in range(999)], 60, tree=False, probs=probs, seed=1))
    check(*draft([2] * 700, 5000, tree=True, probs=False, seed=2))


def test_long_chains():
    for probs in (False, True):
        x, tokens, cu, u, _, q = draft([200, 70, 130], 90, tree=False, probs=probs, seed=3, easy=1.0)
        u[:] = np.minimum(u, 1e-3)  # nearly all are accepted
        u[150] = 0.99999
        got = check(x, tokens, cu, u, None, q)
        assert got.accepted.max() > 64


def test_largest_vocabulary():
    check(*draft([3, 4], 152064, tree=True, probs=False, seed=4))
    check(*draft([3], 152064, tree=False, probs=True, seed=5))


def test_equal_logits_take_the_lowest():
    x = torch.zeros((4, 5000))
    x[1:, 4200] = 1.0
    x[1:, 70] = 1.0
    x[1:, 4999] = 1.0
    check(x, [5, 70, 4200, 70], [0, 2, 4], np.full(4, 0.3, dtype=np.float32), None, None, [0.0, 0.0])
    check(x, [5, 0, 9, 9], [0, 2, 4], np.zeros(4, dtype=np.float32), None, None)


def test_rows_without_a_distribution():
    for bad in (math.nan, math.inf, "nothing"):
        for T in (None, [0.0, 0.0, 1.0]):
            for tree in (False, True):
                x, tokens, cu, u, parents, _ = draft([5, 4, 3], 5000, tree=tree, probs=False, seed=6, easy=1.0)
                u[:] = 1e-3
                for row in (1, 5, 9):
                    if bad == "nothing":
                        x[row] = -math.inf
                    else:
                        x[row, 4321] = bad
                got = check(x, tokens, cu, u, parents, None, T)
                assert -1 in got.next_tokens.tolist()


def test_masked_logits():
    x, tokens, cu, u, parents, _ = draft([5, 9], 5000, tree=True, probs=False, seed=7)
    x[:, ::2] = -math.inf
    x[:, 1::4] = -3.4e38
    tokens = [t | 3 for t in tokens]
    check(x, tokens, cu, u, parents, None)
    x[:, 3::4] = -3.4028234663852886e38  # nothing but the lowest values
    check(x, tokens, cu, u, parents, None)


def test_tokens_that_are_none_and_parents_that_are_none():
    x, tokens, cu, u, parents, _ = draft([8, 8], 300, tree=True, probs=False, seed=8, easy=1.0)
    tokens[1], tokens[3], tokens[9] = -1, 300, 2 ** 31 - 1
    tokens[0] = -5  # (token 0 is known: what it is does not matter)
    parents[4], parents[10], parents[12] = 4, 99, -2 ** 31
    check(x, tokens, cu, u, parents, None)
    x, tokens, cu, u, _, q = draft([6], 300, tree=False, probs=True, seed=9)
    tokens[2] = 301
    u[:3] = 0.001
    check(x, tokens, cu, u, None, q)


def test_the_same_token_twice():
    # refused once it is refused; three children of the root, two alike
    for u1 in (0.01, 0.6, 0.999):
        x = torch.zeros((4, 10))
        x[0, 3] = 1.0
        u = np.float32([0.2, 0.999, u1, u1])
        check(x, [0, 3, 3, 4], [0, 4], u, [-1, 0, 0, 0], None)
        check(x, [0, 3, 3, 4], [0, 4], np.float32([0.9, 0.01, u1, u1]), [-1, 0, 0, 0], None)


def test_all_of_a_distribution_is_refused():
    # children that hold everything, the last refused by its random number all the same
    x = torch.tensor([[5.0, 4.0, -math.inf, -math.inf]] * 3)
    u = np.float32([0.5, 0.99999, 0.99999994])
    check(x, [0, 0, 1], [0, 3], u, [-1, 0, 0], None)
    # draft probabilities equal to the target's: nothing is left
    p = torch.softmax(x.double(), -1).numpy()
    got = step.verify_draft(x.cuda(), ints([0, 0, 1]), ints([0, 3]), torch.tensor([0.5, 2.0, 0.0], device="cuda"),
                            draft_probs=torch.from_numpy(p).float().cuda())
    assert got.accepted.tolist() == [1] and got.next_tokens.tolist()[0] in (0, 1)


def test_uniforms_at_the_ends():
    for u0 in (0.0, 1 - 2.0 ** -24):
        x, tokens, cu, u, _, _ = draft([1] * 9, 9000, tree=False, probs=False, seed=10)
        u[:] = u0
        x[:, -50:] = -math.inf
        check(x, tokens, cu, u, None, None)


@pytest.mark.parametrize("tree, probs", KINDS)
def test_accepted_and_sampled_tokens_have_the_targets_distribution(tree, probs):
    # what follows token 0, accepted or drawn: of 8000 requests with the same rows
    B, V, n = 8000, 6, 4
    g = torch.Generator(device="cuda").manual_seed(11)
    row = torch.tensor([1.0, 0.3, -0.5, 0.0, 1.4, -2.0], device="cuda")
    x = row.expand(B * n, V).contiguous()
    q = torch.softmax(torch.tensor([0.2, 1.0, 0.0, -1.0, 0.5, 0.0], device="cuda"), 0)
    tokens = torch.multinomial(q, B * n, replacement=True, generator=g).int()
    parents = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda").repeat(B) if tree else None
    cu = torch.arange(0, B * n + 1, n, dtype=torch.int32, device="cuda")
    u = torch.rand(B * n, device="cuda", generator=g)
    if not probs:
        tokens = torch.tensor([0, 1, 4, 2], dtype=torch.int32, device="cuda").repeat(B)  # (given, not drawn)
    r = step.verify_draft(x, tokens, cu, u, parents=parents, draft_probs=q.expand(B * n, V).contiguous() if probs else None)
    second = r.path.view(B, n)[:, 1]
    first = torch.where(second < 0, r.next_tokens, tokens.view(B, n).gather(1, second.clamp(min=0)[:, None].long())[:, 0])
    p = torch.softmax(row.double(), 0).cpu()
    count = torch.bincount(first.long(), minlength=V).cpu().double()
    assert bool(((count - B * p).abs() <= 5 * (B * p * (1 - p)).sqrt()).all()), (count / B, p)


def test_refusals():
    x, i, u = torch.zeros((3, 9), device="cuda"), ints([0, 1, 2]), torch.zeros(3, device="cuda")
    cu = ints([0, 3])
    for bad, match in (
            (lambda: step.verify_draft(x.t(), i, cu, u), "contiguous rows"),
            (lambda: step.verify_draft(x.double(), i, cu, u), "fp32, fp16 or bf16"),
            (lambda: step.verify_draft(x, i.long(), cu, u), "tokens"),
            (lambda: step.verify_draft(x, i, cu[:1], u), "cu"),
            (lambda: step.verify_draft(x, i, cu, u.double()), "uniforms"),
            (lambda: step.verify_draft(x, i, cu, u, parents=i[:2]), "parents"),
            (lambda: step.verify_draft(x, i, cu, u, draft_probs=x[:2]), "draft_probs"),
            (lambda: step.verify_draft(x, i, cu, u, draft_probs=x.half()), "draft_probs"),
            (lambda: step.verify_draft(x, i, cu, u, draft_probs=x, parents=i), "chains"),
            (lambda: step.verify_draft(x, i, cu, u, temperature=u), "temperature")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    r = step.verify_draft(x[:0], i[:0], ints([0, 0, 0]), u[:0])
    assert r.accepted.tolist() == [0, 0] and r.next_tokens.tolist() == [-1, -1] and r.path.numel() == 0


# ---------------------------------------------------------------- together

def state_of(seed, window):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    hq, hkv, D, bs = 8, 2, 64, 16
    lengths, new = [700, 0, 33], [9, 4, 1]
    N = sum(new)
    table = torch.zeros((3, 50), dtype=torch.int32)
    table[0, :44] = torch.arange(44)
    table[2, :3] = torch.arange(44, 47)
    parents = sum([[-1] + [int(rng.integers(0, i)) for i in range(1, n)] for n in new], [])
    k, v = step.paged_cache(60, bs, hkv, D, torch.int8)
    for c in (k, v):
        c.codes[:47] = torch.randint(-127, 128, (47, bs, hkv, D), generator=g, dtype=torch.int8).cuda()
        c.scales[:47] = 0.02
    logits = 3 * torch.randn((N, 32000), generator=g).cuda()
    tokens = logits[[0, 0, 0, 1, 1, 2, 3, 4, 4, 9, 9, 10, 11, 13]].topk(2, -1).indices[:, seed % 2].int()
    return [ints(lengths), ints(new), table.cuda(), ints(range(47, 60)), ints(parents),
            torch.randn((N, (hq + 2 * hkv) * D), generator=g).cuda(), step.rope_table(800, D), *k, *v, logits, tokens,
            torch.rand(N, generator=g).cuda()]


def step_of(state, window):
    lengths, new, table, free, parents, x, t, kc, ks, vc, vs, logits, tokens, u = state
    k, v = step.Cache8(kc, ks), step.Cache8(vc, vs)
    plan = step.plan_step(lengths, new, table, free, 16, x.shape[0], parents=parents)
    q = step.qk_norm_rope(x, plan.positions, plan.slots, t, k, v)
    o = step.tree_attention(q, k, v, table, lengths, plan.cu, plan.masks, max_new=9, window=window,
                            sinks=4 if window else 0)
    r = step.verify_draft(logits, tokens, plan.cu, u, parents=parents)
    step.keep_accepted(k, v, table, lengths, plan.cu, r.path, r.accepted)
    kk, vv = step.read_cache(k, v, table, plan.cu, x.shape[0], first=lengths)
    return o, r.accepted, r.path, r.next_tokens, kk, vv


@pytest.mark.parametrize("window", [None, 128])
def test_a_sampled_step_on_another_stream_and_in_a_graph(window):
    state = state_of(1, window)
    want = [t.clone() for t in step_of([t.clone() for t in state], window)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step_of([t.clone() for t in state], window)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with torch.cuda.stream(side):
        step.reserve()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        kept = step_of(state, window)
    for r in range(4):
        other = state_of(2 + r, window)  # new inputs in the same buffers
        for a, b in zip(state, other):
            a.copy_(b)
        fresh = step_of(other, window)  # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(fresh, kept):
            assert torch.equal(a, b), r


def test_steps_on_two_streams_at_once():
    states = [state_of(1, None), state_of(2, None)]
    want = [[t.clone() for t in step_of([t.clone() for t in s], w)] for s, w in zip(states, (None, 128))]
    copies = [[[t.clone() for t in s] for s in states] for _ in range(6)]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for c in copies:
        for i, w in enumerate((None, 128)):
            with torch.cuda.stream(sides[i]):
                got[i].append(step_of(c[i], w))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(want[i], g))


def test_graphs_of_two_streams_at_once():
    states, sides, graphs, kept = [state_of(1, None), state_of(2, None)], [torch.cuda.Stream(), torch.cuda.Stream()], [], []
    want = [[t.clone() for t in step_of([t.clone() for t in s], w)] for s, w in zip(states, (None, 128))]
    for s, side, w in zip(states, sides, (None, 128)):
        with torch.cuda.stream(side):
            step.reserve()
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            kept.append(step_of(s, w))
    fresh = [[t.clone() for t in s] for s in (state_of(1, None), state_of(2, None))]
    for _ in range(4):
        for s, f in zip(states, fresh):
            for a, b in zip(s, f):
                a.copy_(b)
        torch.cuda.synchronize()
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                g.replay()
        torch.cuda.synchronize()
        for k, x in zip(kept, want):
            assert all(torch.equal(a, b) for a, b in zip(k, x))


def test_a_padded_step():
    # buffers longer than the step: rows behind the last request change nothing and come out empty
    state = state_of(3, None)
    lengths, new, table, free, parents, x, rope, kc, ks, vc, vs, logits, tokens, u = state
    want = [t.clone() for t in step_of([t.clone() for t in state], 128)]
    N, more = x.shape[0], 5

    def longer(t, value):
        return torch.cat([t, torch.full((more, *t.shape[1:]), value, dtype=t.dtype, device="cuda")])

    padded = [lengths, new, table, free, longer(parents, -1), longer(x, math.nan), rope, kc, ks, vc, vs,
              longer(logits, math.nan), longer(tokens, 7), longer(u, 0.5)]
    o, accepted, path, following, k, v = step_of(padded, 128)
    for a, b in zip((o[:N], accepted, path[:N], following, k[:N], v[:N]), want):
        assert torch.equal(a, b)
    assert not o[N:].any() and bool((path[N:] == -1).all()) and not k[N:].any() and not v[N:].any()


def test_no_tokens_at_all():
    k, v = step.paged_cache(4, 16, 2, 64, torch.int8)
    table, none, cu = ints([[0, 1], [2, 3]]), ints([]), ints([0, 0, 0])
    q = step.qk_norm_rope(torch.zeros((0, 8 * 64), device="cuda"), none, none, step.rope_table(8, 64), k, v)
    assert tuple(q.shape) == (0, 4, 64)
    for window in (None, 8):
        assert step.tree_attention(q, k, v, table, ints([5, 0]), cu, window=window).numel() == 0
    step.keep_accepted(k, v, table, ints([5, 0]), cu, none, ints([0, 0]))
    kk, vv = step.read_cache(k, v, table, cu, 0)
    assert kk.numel() == 0 and vv.numel() == 0


def test_capture_without_a_workspace_is_refused():
    from forge_amd import _lib
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert _lib.lib().fq_release_workspace(side.cuda_stream) == 0  # (streams are reused)
    x, i, u, cu = torch.zeros((3, 9), device="cuda"), ints([0, 1, 2]), torch.zeros(3, device="cuda"), ints([0, 3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        with pytest.raises(_lib.FqError, match="workspace"):
            step.verify_draft(x, i, cu, u)


def test_sample_drafts_example(capsys):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "sample_drafts.py")
    runpy.run_path(path)["main"]()
    out = capsys.readouterr().out
    assert "tokens" in out and "8 bits" in out
