"""CPU tests of include/forge_step.h's entry points: arguments are refused before
a device is touched, empty calls do nothing."""
from __future__ import annotations

import ctypes

import pytest
import torch

from forge_amd import _lib, step

P = ctypes.c_void_p(4096)  # never read: the checks come first
F16, F32, BF16 = 1, 0, 100


def plan(**k):
    a = dict(lengths=P, new=P, parents=None, B=2, N=4, bs=16, table=P, cols=3, stride=3, free=P,
             n_free=5, cu=P, slots=P, positions=P, masks=None, info=P)
    a.update(k)
    return _lib.lib().fq_plan_step(*a.values(), None)


@pytest.mark.parametrize("k, want", [
    (dict(B=0), _lib.FQ_ERR_SHAPE), (dict(B=8193), _lib.FQ_ERR_SHAPE), (dict(N=-1), _lib.FQ_ERR_SHAPE),
    (dict(bs=8), _lib.FQ_ERR_SHAPE), (dict(bs=24), _lib.FQ_ERR_SHAPE), (dict(bs=2048), _lib.FQ_ERR_SHAPE),
    (dict(cols=0), _lib.FQ_ERR_SHAPE), (dict(stride=2), _lib.FQ_ERR_SHAPE), (dict(n_free=-1), _lib.FQ_ERR_SHAPE),
    (dict(lengths=None), _lib.FQ_ERR_NULL), (dict(free=None), _lib.FQ_ERR_NULL),
    (dict(slots=None), _lib.FQ_ERR_NULL), (dict(parents=P), _lib.FQ_ERR_NULL), (dict(info=None), _lib.FQ_ERR_NULL)])
def test_plan_refuses(k, want):
    assert plan(**k) == want


CACHE = dict(type=F16, k=P, v=P, nb=4, bs=16, sb=16 * 2 * 64, st=2 * 64, sh=64)
BAD_CACHE = [(dict(type=F32), _lib.FQ_ERR_DTYPE), (dict(type=7), _lib.FQ_ERR_DTYPE), (dict(nb=0), _lib.FQ_ERR_SHAPE),
             (dict(bs=20), _lib.FQ_ERR_SHAPE), (dict(nb=2 ** 28), _lib.FQ_ERR_SHAPE), (dict(st=-8), _lib.FQ_ERR_SHAPE),
             (dict(k=None), _lib.FQ_ERR_NULL), (dict(v=None), _lib.FQ_ERR_NULL),
             (dict(k=ctypes.c_void_p(8)), _lib.FQ_ERR_ALIGN), (dict(sh=68), _lib.FQ_ERR_ALIGN)]


def rope(N=2, ld=512, hq=4, hkv=2, D=64, rot=64, qkv=P, table=P, rows=100, q=P, **c):
    c = {**CACHE, **c}
    return _lib.lib().fq_qk_norm_rope(qkv, ld, N, hq, hkv, D, rot, 0, None, None, None, 1e-6, P, P,
                                      table, rows, q, *c.values(), None)


@pytest.mark.parametrize("k, want", BAD_CACHE + [
    (dict(N=-1), _lib.FQ_ERR_SHAPE), (dict(hq=3), _lib.FQ_ERR_SHAPE), (dict(hkv=0), _lib.FQ_ERR_SHAPE),
    (dict(D=60), _lib.FQ_ERR_SHAPE), (dict(D=520), _lib.FQ_ERR_SHAPE), (dict(rot=72), _lib.FQ_ERR_SHAPE),
    (dict(rot=12), _lib.FQ_ERR_SHAPE), (dict(ld=511), _lib.FQ_ERR_SHAPE), (dict(N=2 ** 25), _lib.FQ_ERR_SHAPE),
    (dict(qkv=None), _lib.FQ_ERR_NULL), (dict(table=None), _lib.FQ_ERR_NULL), (dict(q=None), _lib.FQ_ERR_NULL),
    (dict(N=0), _lib.FQ_OK)])
def test_rope_refuses(k, want):
    assert rope(**k) == want


def attention(q=P, ldq=256, B=1, N=2, new=2, hq=4, hkv=2, D=64, table=P, cols=3, stride=3, out=P, **c):
    c = {**CACHE, **c}
    return _lib.lib().fq_tree_attention(q, ldq, P, P, None, B, N, new, hq, hkv, D, 0.1, *c.values(),
                                        table, cols, stride, out, None)


@pytest.mark.parametrize("k, want", BAD_CACHE + [
    (dict(B=0), _lib.FQ_ERR_SHAPE), (dict(N=-1), _lib.FQ_ERR_SHAPE), (dict(new=-1), _lib.FQ_ERR_SHAPE),
    (dict(hq=5), _lib.FQ_ERR_SHAPE), (dict(D=80), _lib.FQ_ERR_SHAPE), (dict(D=512), _lib.FQ_ERR_SHAPE),
    (dict(ldq=255), _lib.FQ_ERR_SHAPE), (dict(cols=0), _lib.FQ_ERR_SHAPE), (dict(stride=1), _lib.FQ_ERR_SHAPE),
    (dict(q=None), _lib.FQ_ERR_NULL), (dict(table=None), _lib.FQ_ERR_NULL), (dict(out=None), _lib.FQ_ERR_NULL),
    (dict(out=ctypes.c_void_p(4100)), _lib.FQ_ERR_ALIGN), (dict(N=0), _lib.FQ_OK)])
def test_attention_refuses(k, want):
    assert attention(**k) == want


def logprobs(x=P, type=F32, ld=100, M=2, V=100, targets=P, J=1, top=5, lp=P, H=P, tl=P, tt=P):
    return _lib.lib().fq_token_logprobs(x, type, ld, M, V, targets, J, top, lp, H, tl, tt, None)


@pytest.mark.parametrize("k, want", [
    (dict(type=2), _lib.FQ_ERR_DTYPE), (dict(M=-1), _lib.FQ_ERR_SHAPE), (dict(V=0), _lib.FQ_ERR_SHAPE),
    (dict(V=2 ** 30 + 1, ld=2 ** 31), _lib.FQ_ERR_SHAPE), (dict(ld=99), _lib.FQ_ERR_SHAPE),
    (dict(J=-1), _lib.FQ_ERR_SHAPE), (dict(top=65), _lib.FQ_ERR_SHAPE), (dict(V=4, top=5), _lib.FQ_ERR_SHAPE),
    (dict(x=None), _lib.FQ_ERR_NULL), (dict(targets=None), _lib.FQ_ERR_NULL), (dict(tt=None), _lib.FQ_ERR_NULL),
    (dict(x=ctypes.c_void_p(4098)), _lib.FQ_ERR_ALIGN), (dict(M=0), _lib.FQ_OK)])
def test_logprobs_refuses(k, want):
    assert logprobs(**k) == want


def test_host_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    k = torch.zeros(2, 16, 1, 64, dtype=torch.float16)
    t = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: step.plan_step(i, i, t, i, 16, 2),
                 lambda: step.qk_norm_rope(torch.zeros(2, 192), i, i, torch.zeros(4, 64), k, k),
                 lambda: step.tree_attention(torch.zeros(2, 1, 64), k, k, t, i, torch.zeros(3, dtype=torch.int32)),
                 lambda: step.token_logprobs(torch.zeros(2, 9))):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()


def test_paged_cache_is_laid_out_by_head():
    k, v = step.paged_cache(3, 32, 2, 64, torch.bfloat16, device="cpu")
    assert k.shape == v.shape == (3, 32, 2, 64) and k.dtype == torch.bfloat16
    assert k.stride() == (32 * 2 * 64, 64, 32 * 64, 1) and not k.any()


def test_rope_table():
    t = step.rope_table(5, 8, base=100.0, device="cpu")
    assert t.shape == (5, 8)
    a = 3 * torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64)
    assert torch.allclose(t[3].double(), torch.cat([a.cos(), a.sin()]), atol=1e-7)
