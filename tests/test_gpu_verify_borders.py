"""verify_draft where a random number lies next to the border of acceptance: the fp32 numbers on
either side of it, against probabilities in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from forge_amd import step

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


def around(border):
    """The largest fp32 below the border (in 64 bits) and the smallest above it."""
    u = np.float32(border)
    low = u if float(u) < border else np.nextafter(u, np.float32(0))
    return low, np.nextafter(low, np.float32(2))


def clear(border):
    """Whether both are 2^-28 of the border away from it and more.  (What sums in 64 bits are off by,
    2^-50, is 2^-30 of what is left where that is 1e-6 of them.)"""
    low, high = around(border)
    return min(border - float(low), float(high) - border) > 2.0 ** -28 * border and float(high) < 1


def softmax(x, T):
    e = np.exp((x - x.max()) / np.float64(np.float32(T)))
    return e / e.sum()


@pytest.mark.parametrize("V, dtype, T", [(17, torch.float32, 1.0), (1000, torch.float32, 0.7), (32000, torch.float32, 0.7),
                                         (32000, torch.bfloat16, 1.3), (152064, torch.float32, 0.7), (152064, torch.float16, 1.0)])
@pytest.mark.parametrize("probs", [False, True])
def test_chains(V, dtype, T, probs):
    rng = np.random.default_rng(V)
    B = 24
    x = torch.from_numpy(2.0 * rng.standard_normal((2 * B, V))).to(dtype)
    tokens, u = np.zeros(2 * B, dtype=np.int32), np.full(2 * B, 0.5, dtype=np.float32)
    q = torch.from_numpy(rng.random((2 * B, V))).float() if probs else None
    want = []
    for b in range(B):
        p = softmax(x[2 * b].double().numpy(), T)
        t = int(p.argmax())
        while True:
            border = p[t]
            if probs:  # u q < p
                q[2 * b + 1, t] = min(1.0, float(rng.uniform(1.1, 3)) * p[t])
                border = p[t] / float(q[2 * b + 1, t])
            if clear(border):
                break
            t = int(rng.integers(V))
        low, high = around(border)
        tokens[2 * b + 1], u[2 * b + 1] = t, (low, high)[b % 2]
        want.append(2 if b % 2 == 0 else 1)
    done = step.verify_draft(x.cuda(), ints(tokens), ints(np.arange(B + 1) * 2), torch.from_numpy(u).cuda(),
                             draft_probs=None if q is None else q.cuda(), temperature=torch.full((B,), T, device="cuda"))
    assert done.accepted.tolist() == want


@pytest.mark.parametrize("V, T", [(40, 1.0), (32000, 0.7), (152064, 1.0)])
@pytest.mark.parametrize("rest", [0.3, 1e-2, 1e-4, 1e-6])
def test_siblings_that_hold_nearly_all(V, T, rest):
    """Two refused siblings leave `rest` of the distribution; the third one's border is its share of that."""
    rng = np.random.default_rng(V)
    B = 24
    x = 0.5 * rng.standard_normal((4 * B, V))
    tokens, u = np.zeros(4 * B, dtype=np.int32), np.full(4 * B, 0.5, dtype=np.float32)
    parents = np.tile([-1, 0, 0, 0], B)
    xs = torch.empty((4 * B, V))
    want = []
    for b in range(B):
        row = x[4 * b]
        a, c = rng.choice(V, 2, replace=False)
        others = np.delete(row, [a, c])
        whole = np.exp(others / T).sum()
        row[a] = T * np.log(0.6 * whole * (1 - rest) / rest)
        row[c] = T * np.log(0.4 * whole * (1 - rest) / rest)
        xs[4 * b:4 * b + 4] = torch.from_numpy(x[4 * b:4 * b + 4]).float()
        e = np.exp((xs[4 * b].double().numpy() - float(xs[4 * b].max())) / np.float64(np.float32(T)))
        p = e / e.sum()
        left = np.delete(e, [a, c]).sum() / e.sum()  # (not one less the others: no bits are lost)
        t = a
        while t in (a, c) or not clear(e[t] / np.delete(e, [a, c]).sum()):
            t = rng.integers(V)
        low, high = around(e[t] / np.delete(e, [a, c]).sum())
        tokens[4 * b + 1:4 * b + 4] = a, c, t
        # the first two are refused: above their own borders
        u[4 * b + 1] = min(np.float32(p[a] * 1.0001) + np.float32(1e-6), np.float32(1 - 2.0 ** -24))
        u[4 * b + 2] = min(np.float32(p[c] / (1 - p[a]) * 1.0001) + np.float32(1e-6), np.float32(1 - 2.0 ** -24))
        assert u[4 * b + 1] > p[a] and u[4 * b + 2] > p[c] / (p[c] + left)
        u[4 * b + 3] = (low, high)[b % 2]
        want.append(2 if b % 2 == 0 else 1)
    done = step.verify_draft(xs.cuda(), ints(tokens), ints(np.arange(B + 1) * 4), torch.from_numpy(u).cuda(),
                             parents=ints(parents), temperature=torch.full((B,), T, device="cuda"))
    assert done.accepted.tolist() == want


def test_a_deep_branch_of_borders():
    """Each token of a branch next to its border, below it but for the last, behind refused siblings here and there."""
    V, n, T = 5000, 30, 0.9
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((2 * n + 1, V))).float()
    tokens, u, parents = [0], [0.5], [-1]
    last = 0
    for d in range(n):
        p = softmax(x[last].double().numpy(), T)
        t = int(p.argmax())
        low, high = around(p[t])
        at = len(tokens)
        # (a sibling of no probability to speak of first in every third)
        if d % 3 == 0:
            tokens.append(int(p.argmin())), u.append(0.999), parents.append(last)
            mass = 1 - p[tokens[-1]]
            low, high = around(p[t] / mass)
            at += 1
        tokens.append(t), u.append(low if d < n - 1 else high), parents.append(last)
        last = at if d < n - 1 else last
    N = len(tokens)
    done = step.verify_draft(x[:N].cuda(), ints(tokens), ints([0, N]), torch.tensor(np.asarray(u, dtype=np.float32), device="cuda"),
                             parents=ints(parents), temperature=torch.tensor([T], device="cuda"))
    assert done.accepted.tolist() == [n]
    assert done.path.tolist()[n - 1] == last


@pytest.mark.parametrize("n", [64, 65, 140])
def test_long_chains_of_borders(n):
    """Two chains, each token next to its border: one accepted to its end, one but for its last token."""
    V, T = 700, 1.1
    rng = np.random.default_rng(n)
    x = torch.from_numpy(1.5 * rng.standard_normal((2 * n, V))).float()
    tokens, u = np.zeros(2 * n, dtype=np.int32), np.full(2 * n, 0.5, dtype=np.float32)
    for i in range(2 * n):
        if i % n:
            p = softmax(x[i - 1].double().numpy(), T)
            tokens[i] = t = next(int(t) for t in np.argsort(-p) if clear(p[t]))
            u[i] = around(p[t])[i == 2 * n - 1]
    done = step.verify_draft(x.cuda(), ints(tokens), ints([0, n, 2 * n]), torch.from_numpy(u).cuda(),
                             temperature=torch.full((2,), T, device="cuda"))
    assert done.accepted.tolist() == [n, n - 1]
    assert done.path.tolist() == list(range(n)) + list(range(n - 1)) + [-1]


@pytest.mark.parametrize("T", [2.0 ** -130, 2.0 ** -120, 2.0 ** 110, 2.0 ** 126])
def test_temperatures_far_out(T):
    """Temperatures whose inverse, or whose logits' differences, leave fp32's range."""
    V = 300
    rng = np.random.default_rng(8)
    x = (0.9 * rng.standard_normal((16, V)) * T).astype(np.float32)
    tokens, u, want = np.zeros(16, dtype=np.int32), np.full(16, 0.5, dtype=np.float32), []
    for b in range(8):
        p = softmax(x[2 * b].astype(np.float64), T)
        tokens[2 * b + 1] = t = int(p.argmax())
        u[2 * b + 1] = around(p[t])[b % 2]
        want.append(2 if b % 2 == 0 else 1)
    done = step.verify_draft(torch.from_numpy(x).cuda(), ints(tokens), ints(np.arange(9) * 2), torch.from_numpy(u).cuda(),
                             temperature=torch.full((8,), T, device="cuda"))
    assert done.accepted.tolist() == want
