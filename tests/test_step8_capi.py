"""CPU tests of include/forge_step.h's entry points for caches of 8 bits, windows and drafts:
arguments are refused before a device is touched, empty calls do nothing."""
from __future__ import annotations

import ctypes

import pytest
import torch

from forge_amd import _lib, step

P = ctypes.c_void_p(4096)  # never read: the checks come first
F16, F32, BF16, I8 = 1, 0, 100, 101
DTYPE, SHAPE, NULL, ALIGN, OK = (_lib.FQ_ERR_DTYPE, _lib.FQ_ERR_SHAPE, _lib.FQ_ERR_NULL, _lib.FQ_ERR_ALIGN, _lib.FQ_OK)

CODES = dict(k=P, v=P, ks=P, vs=P, nb=4, bs=16)
STRIDES = dict(sb=16 * 2 * 64, st=2 * 64, sh=64)
BAD_CODES = [(dict(nb=0), SHAPE), (dict(bs=20), SHAPE), (dict(bs=8), SHAPE), (dict(bs=2048), SHAPE), (dict(nb=2 ** 28), SHAPE),
             (dict(st=-16), SHAPE), (dict(st=2 ** 27), SHAPE), (dict(k=None), NULL), (dict(v=None), NULL), (dict(ks=None), NULL),
             (dict(vs=None), NULL), (dict(k=ctypes.c_void_p(8)), ALIGN), (dict(ks=ctypes.c_void_p(4098)), ALIGN),
             (dict(sh=72), ALIGN)]


def rope8(N=2, ld=512, hq=4, hkv=2, D=64, rot=64, qkv=P, table=P, rows=100, q=P, **c):
    c = {**CODES, **STRIDES, **c}
    return _lib.lib().fq_qk_norm_rope8(qkv, ld, N, hq, hkv, D, rot, 0, None, None, None, 1e-6, P, P,
                                       table, rows, q, *c.values(), None)


@pytest.mark.parametrize("k, want", BAD_CODES + [
    (dict(N=-1), SHAPE), (dict(hq=3), SHAPE), (dict(D=72, ld=9999), SHAPE), (dict(D=528, ld=9999), SHAPE), (dict(rot=12), SHAPE),
    (dict(ld=511), SHAPE), (dict(N=2 ** 25), SHAPE), (dict(qkv=None), NULL), (dict(table=None), NULL), (dict(q=None), NULL),
    (dict(N=0), OK)])
def test_rope8_refuses(k, want):
    assert rope8(**k) == want


def read(hkv=2, D=64, table=P, cols=3, stride=3, starts=P, B=2, N=4, type=F16, ko=P, vo=P, **c):
    c = {**CODES, **c}
    s = {n: c.pop(n, d) for n, d in STRIDES.items()}
    return _lib.lib().fq_read_cache8(*c.values(), hkv, D, *s.values(), table, cols, stride, starts, None, B, N, type, ko, vo, None)


@pytest.mark.parametrize("k, want", BAD_CODES + [
    (dict(hkv=0), SHAPE), (dict(D=72), SHAPE), (dict(D=528), SHAPE), (dict(hkv=2 ** 20), SHAPE), (dict(cols=0), SHAPE),
    (dict(stride=2), SHAPE), (dict(B=0), SHAPE), (dict(N=-1), SHAPE), (dict(type=I8), DTYPE), (dict(table=None), NULL),
    (dict(starts=None), NULL), (dict(ko=None), NULL), (dict(vo=ctypes.c_void_p(4104)), ALIGN), (dict(N=0), OK)])
def test_read_refuses(k, want):
    assert read(**k) == want


def attention(q=P, ldq=256, B=1, N=2, new=2, hq=4, hkv=2, D=64, window=5, sinks=1, type=I8, table=P, cols=3, stride=3, out=P, **c):
    c = {**CODES, **STRIDES, **c}
    return _lib.lib().fq_window_attention(q, ldq, P, P, None, B, N, new, hq, hkv, D, 0.1, window, sinks, type, *c.values(),
                                          table, cols, stride, out, None)


@pytest.mark.parametrize("k, want", BAD_CODES + [
    (dict(B=0), SHAPE), (dict(N=-1), SHAPE), (dict(new=-1), SHAPE), (dict(hq=5), SHAPE), (dict(D=80), SHAPE), (dict(D=512), SHAPE),
    (dict(ldq=255), SHAPE), (dict(cols=0), SHAPE), (dict(stride=1), SHAPE), (dict(window=-1), SHAPE), (dict(sinks=-1), SHAPE),
    (dict(type=F32), DTYPE), (dict(q=None), NULL), (dict(table=None), NULL), (dict(out=None), NULL),
    (dict(out=ctypes.c_void_p(4100)), ALIGN), (dict(N=0), OK), (dict(type=F16, ks=None, vs=None, N=0), OK),
    (dict(type=BF16, sh=68), ALIGN)])
def test_window_attention_refuses(k, want):
    assert attention(**k) == want


def test_tree_attention_takes_no_codes():
    assert _lib.lib().fq_tree_attention(P, 256, P, P, None, 1, 2, 2, 4, 2, 64, 0.1, I8, P, P, 4, 16, 2048, 128, 64, P, 3, 3,
                                        P, None) == DTYPE


def verify(x=P, type=F32, ld=100, V=100, tokens=P, cu=P, B=2, N=4, parents=None, u=P, q=None, ldp=100, acc=P, path=P, nxt=P):
    return _lib.lib().fq_verify_draft(x, type, ld, V, tokens, cu, B, N, parents, u, q, ldp, None, acc, path, nxt, None)


@pytest.mark.parametrize("k, want", [
    (dict(type=2), DTYPE), (dict(B=0), SHAPE), (dict(B=8193), SHAPE), (dict(N=-1), SHAPE), (dict(N=2 ** 20 + 1), SHAPE),
    (dict(V=0), SHAPE), (dict(V=2 ** 30 + 1, ld=2 ** 31), SHAPE), (dict(ld=99), SHAPE), (dict(q=P, ldp=99), SHAPE),
    (dict(q=P, parents=P), SHAPE), (dict(cu=None), NULL), (dict(acc=None), NULL), (dict(nxt=None), NULL), (dict(x=None), NULL),
    (dict(tokens=None), NULL), (dict(u=None), NULL), (dict(path=None), NULL), (dict(x=ctypes.c_void_p(4098)), ALIGN)])
def test_verify_refuses(k, want):
    assert verify(**k) == want


def keep(type=I8, hkv=2, D=64, table=P, cols=3, stride=3, lengths=P, cu=P, path=P, acc=P, B=2, N=4, **c):
    c = {**CODES, **c}
    s = {n: c.pop(n, d) for n, d in STRIDES.items()}
    return _lib.lib().fq_keep_accepted(type, *c.values(), hkv, D, *s.values(), table, cols, stride, lengths, cu, path, acc,
                                       B, N, None)


@pytest.mark.parametrize("k, want", BAD_CODES + [
    (dict(type=F32), DTYPE), (dict(hkv=0), SHAPE), (dict(D=72), SHAPE), (dict(D=528), SHAPE), (dict(B=2 ** 23 + 1), SHAPE),
    (dict(cols=0), SHAPE), (dict(stride=2), SHAPE), (dict(B=0), SHAPE), (dict(N=-1), SHAPE), (dict(table=None), NULL),
    (dict(lengths=None), NULL), (dict(cu=None), NULL), (dict(path=None), NULL), (dict(acc=None), NULL), (dict(N=0), OK),
    (dict(type=BF16, ks=None, vs=None, N=0), OK), (dict(type=F16, D=60), SHAPE), (dict(type=F16, sh=68), ALIGN)])
def test_keep_refuses(k, want):
    assert keep(**k) == want


def test_paged_cache_of_8_bits():
    k, v = step.paged_cache(3, 32, 2, 64, torch.int8, device="cpu")
    assert k.codes.shape == v.codes.shape == (3, 32, 2, 64) and k.codes.dtype == torch.int8
    assert k.codes.stride() == (32 * 2 * 64, 64, 32 * 64, 1) and not k.codes.any()
    assert k.scales.shape == (3, 2, 2) and k.scales.dtype == torch.float32 and not k.scales.any()


def test_host_tensors_are_refused():
    i = torch.zeros(2, dtype=torch.int32)
    k, v = step.paged_cache(2, 16, 1, 64, torch.int8, device="cpu")
    t = torch.zeros(2, 1, dtype=torch.int32)
    for call in (lambda: step.read_cache(k, v, t, torch.zeros(3, dtype=torch.int32), 2),
                 lambda: step.keep_accepted(k, v, t, i, torch.zeros(3, dtype=torch.int32), i, i),
                 lambda: step.verify_draft(torch.zeros(2, 9), i, i, torch.zeros(2))):
        with pytest.raises(RuntimeError, match="device tensor"):
            call()


@pytest.mark.parametrize("call", [
    lambda: keep(B=2 ** 22, hkv=2), lambda: keep(B=2 ** 23, hkv=1), lambda: keep(type=F16, ks=None, vs=None, B=2 ** 23, hkv=1),
    lambda: read(hkv=1, D=16, N=2 ** 28), lambda: read(hkv=1, D=16, N=2 ** 31 - 1), lambda: read(hkv=64, D=512, N=2 ** 24)])
def test_grids_of_more_lanes_than_32_bits_are_refused(call):
    assert call() == SHAPE
