"""More operators of a serving step over a paged cache, measured through
forge_amd.step: the cache in 8 bits, windows, and the two ends of a verified draft.

A case is one operator:

  attention  tree_attention over a cache of 8-bit codes with a scale for each 16
             tokens and key head
  window     tree_attention with a sliding window and a few first tokens that
             stay visible, over either kind of cache
  write      qk_norm_rope into such a cache of 8 bits, and read_cache of what the
             requests then hold
  verify     verify_draft: drafted tokens against the target's probabilities, from
             given random numbers
  keep       keep_accepted: the accepted branch's keys and values to the slots behind
             the context

Heads: 32 query and 4 key heads of 64 (a small model, hidden 2048), 28 and 4 of
128 (7B, hidden 3584), 32 and 8 of 128 (8B, hidden 4096), and generic ones.
`own` false computes the operators from elementary torch operations in 32 bits
(64 for what a random number is compared with); `own` true calls forge_amd.step.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_ROPE_TABLE = 32768  # positions of the rotation table that a program keeps
_GROUP = 16          # tokens that share a scale


def listed():
    return [
        # one request of a small model, a short chain of drafted tokens: latency
        dict(name="attention, one short chain", op="attention", B=1, ctx=333, T=4, tree=False,
             hq=32, hkv=4, D=64, block=16, cache="i8", window=0, sinks=0),
        # a batch that decodes one token each, 7B heads (7 query heads a key head)
        dict(name="attention, decode batch", op="attention", B=48, ctx=5001, T=1, tree=False,
             hq=28, hkv=4, D=128, block=16, cache="i8", window=0, sinks=0),
        # one long document: the context is split over the whole card
        dict(name="attention, long context", op="attention", B=1, ctx=131000, T=13, tree=True,
             hq=28, hkv=4, D=128, block=64, cache="i8", window=0, sinks=0),
        # a full batch of large trees: the largest attention call
        dict(name="attention, full batch", op="attention", B=32, ctx=8190, T=32, tree=True,
             hq=32, hkv=8, D=128, block=32, cache="i8", window=0, sinks=0),
        # long conversations of a model with windows, one token each
        dict(name="window, decode batch", op="window", B=64, ctx=20001, T=1, tree=False,
             hq=32, hkv=8, D=128, block=32, cache="i8", window=1023, sinks=4),
        # the same with drafted trees and a cache of 16 bits
        dict(name="window, trees", op="window", B=16, ctx=30000, T=9, tree=True,
             hq=28, hkv=4, D=128, block=16, cache="bf16", window=4096, sinks=5),
        # one decoded token of a small model: latency
        dict(name="write, one token", op="write", B=1, ctx=41, T=1, hq=32, hkv=4, D=64, rot=64,
             block=16, bias=False, norm=False, interleaved=True),
        # prompts behind a short beginning, normalized heads: bandwidth
        dict(name="write, prompts", op="write", B=3, ctx=7, T=2731, hq=32, hkv=8, D=128, rot=128,
             block=32, bias=False, norm=True, interleaved=False),
        # one request's chain, drafted by a small model whose probabilities are known
        dict(name="verify, one chain", op="verify", B=1, T=6, V=32000, tree=False, probs=True,
             type="f32", temperature=1.0),
        # a full batch of trees over the largest vocabulary
        dict(name="verify, full batch", op="verify", B=32, T=25, V=152064, tree=True, probs=False,
             type="f32", temperature=0.8),
        # a few requests with drafted trees over a cache of 16 bits
        dict(name="keep, few trees", op="keep", B=7, ctx=150, T=25, hkv=4, D=128, block=16, cache="f16"),
        # a large batch over a cache of 8 bits
        dict(name="keep, large batch", op="keep", B=96, ctx=301, T=48, hkv=8, D=128, block=32, cache="i8"),
    ]


_HEADS = [(32, 4, 64), (28, 4, 128), (32, 8, 128), (12, 12, 64), (9, 3, 96), (10, 2, 256), (5, 1, 128)]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, no
    larger than the largest listed case of its operator."""
    op = rng.choice(["attention", "attention", "window", "write", "verify", "keep"])
    block = rng.choice([16, 32, 64, 128])
    hq, hkv, D = rng.choice(_HEADS)
    if op in ("attention", "window"):
        tree = rng.random() < 0.6
        B, T = _log(rng, 1, 64), _log(rng, 1, 64)
        most = min(131072, 32 * 8190 * 8 * 128 // (B * hkv * D), 32 * 32 * 32 * 8190 // (B * T * hq))
        windowed = op == "window"
        return dict(op=op, B=B, ctx=_log(rng, 1, max(1, most)), T=T, tree=tree, hq=hq, hkv=hkv, D=D,
                    block=block, cache=rng.choice(["i8", "f16", "bf16"]) if windowed else "i8",
                    window=_log(rng, 1, 8192) if windowed else 0,
                    sinks=rng.choice([0, 1, 4, 4, 16, 100]) if windowed else 0)
    if op == "write":
        T = _log(rng, 1, 2731)
        most = 2 * 2731 * 48 * 128 // ((hq + 2 * hkv) * D)
        B = _log(rng, 1, max(1, min(200, most // T)))
        return dict(op=op, B=B, ctx=_log(rng, 1, max(1, min(400, most // B))), T=min(T, most), hq=hq, hkv=hkv,
                    D=D, rot=rng.choice([D, D, D // 2]), block=block, bias=rng.random() < 0.3,
                    norm=rng.random() < 0.5, interleaved=rng.random() < 0.3)
    if op == "verify":
        V, tree = _log(rng, 1000, 200000), rng.random() < 0.5
        T = _log(rng, 1, 64)
        return dict(op=op, B=_log(rng, 1, max(1, min(200, 32 * 25 * 152064 // (3 * T * V)))), T=T, V=V,
                    tree=tree, probs=not tree and rng.random() < 0.6,
                    type=rng.choice(["f32", "f32", "f16", "bf16"]),
                    temperature=rng.choice([1.0, 1.0, 0.7, 1.3, 0.0]))
    return dict(op=op, B=_log(rng, 1, 96), ctx=_log(rng, 1, 301), T=_log(rng, 1, 48), hkv=hkv, D=D,
                block=block, cache=rng.choice(["i8", "f16", "bf16"]))


def _ragged(case):
    """Cached and new tokens of each request: the first has the case's own
    numbers, the others between half of them and them (new tokens: between one
    and them), and of four requests and more the third has nothing cached."""
    def part(b):
        return (b * 0.6180339887498949) % 1.0
    ctx = [case["ctx"] - int(part(b) * (case["ctx"] // 2 + 1)) for b in range(case["B"])]
    new = [max(1, case["T"] - int(part(3 * b) * case["T"])) for b in range(case["B"])]
    if case["B"] >= 4:
        ctx[2] = 0
    return ctx, new


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _starts(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _tree(new, g, dev):
    """Parents [N] of random trees under each request's first token: token i hangs
    on one of the tokens before it."""
    i = torch.cat([torch.arange(n) for n in new]).to(dev)
    r = torch.rand(i.shape, generator=g, device=dev)
    return torch.minimum(torch.floor(r.sqrt() * i).to(torch.int32), i.to(torch.int32) - 1)


def _masks64(parents, new):
    """Bit j of masks[i]: token j of i's request is i or one that i descends from."""
    out, at, p = [], 0, parents.tolist()
    for n in new:
        m = []
        for i in range(n):
            m.append((1 << i) | (m[p[at + i]] if p[at + i] >= 0 else 0))
        out += m
        at += n
    return torch.tensor([v - (1 << 64) if v >> 63 else v for v in out], dtype=torch.int64,
                        device=parents.device)


def _cache8(normal, n, hkv, bs, D):
    """Codes and scales of n blocks of normal keys (a few channels strong, as keys have them)."""
    x = normal(n, hkv, bs, D)
    x[..., ::31] *= 3
    s = x.view(n, hkv, bs // _GROUP, -1).abs().amax(-1) / 127
    c = torch.round(x.view(n, hkv, bs // _GROUP, -1) / s[..., None]).to(torch.int8)
    return c.view(n, hkv, bs, D).transpose(1, 2), s


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    op = case["op"]
    s = dict(op=op, case=case)
    if op == "verify":
        return _prepare_verify(s, case, g, dev, normal)
    ctx, new = _ragged(case)
    cu, bs, hkv, D = _starts(new), case["block"], case["hkv"], case["D"]
    keys = [c + n for c, n in zip(ctx, new)]
    pages = [-(-k // bs) for k in keys]
    n = sum(pages)
    blocks = torch.randperm(n, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((case["B"], max(pages)), dtype=torch.int32, device=dev)
    table[torch.arange(max(pages), device=dev)[None] < _ints(pages, dev)[:, None]] = blocks
    starts = _starts(keys)
    s.update(N=cu[-1], T=max(new), L=max(keys), lengths=_ints(ctx, dev), cu=_ints(cu, dev), table=table,
             starts=_ints(starts, dev), held=starts[-1])
    if op == "write" or case["cache"] == "i8":
        (s["k"], s["ks"]), (s["v"], s["vs"]) = (_cache8(normal, n, hkv, bs, D) for _ in range(2))
    else:
        # a block's rows lie head by head, as paged_cache() lays them out
        s["k"], s["v"] = (normal(n, hkv, bs, D).to(_TYPES[case["cache"]]).transpose(1, 2)
                          for _ in range(2))
    if op in ("attention", "window"):
        s.update(q=2 * normal(cu[-1], case["hq"], D),
                 masks=_masks64(_tree(new, g, dev), new) if case["tree"] else None)
        return s
    if op == "keep":
        # a branch of each request's tree: its first token and some later ones
        i = torch.cat([torch.arange(m) for m in new]).to(dev)
        taken = (torch.rand(i.shape, generator=g, device=dev) < 0.3) | (i == 0)
        first = s["cu"].long()[:-1].repeat_interleave(_ints(new, dev).long())
        rank = taken.long().cumsum(0)
        rank = rank - rank[first]
        path = torch.full((cu[-1],), -1, dtype=torch.int32, device=dev)
        path[(first + rank)[taken]] = i[taken].int()
        s.update(path=path, accepted=torch.zeros(case["B"], dtype=torch.int32, device=dev).index_add_(
            0, torch.arange(case["B"], device=dev).repeat_interleave(_ints(new, dev).long()), taken.int()))
        return s
    N, hq, rot = cu[-1], case["hq"], case["rot"]
    rows = (hq + 2 * hkv) * D
    x = normal(N, rows)
    x[:, ::61] *= 6  # a few strong channels, as projections have them
    angle = torch.arange(_ROPE_TABLE, device=dev, dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
    b = torch.arange(case["B"], device=dev).repeat_interleave(_ints(new, dev).long())
    number = torch.cat([torch.arange(c, c + m) for c, m in zip(ctx, new)]).to(dev)
    slots = table[b, number // bs] * bs + (number % bs).int()
    s.update(qkv=x, rope=torch.cat([angle.cos(), angle.sin()], 1).float(), positions=number.int(),
             slots=slots, bias=normal(rows) if case["bias"] else None,
             qw=1 + 0.2 * normal(D) if case["norm"] else None,
             kw=1 + 0.2 * normal(D) if case["norm"] else None)
    return s


def _prepare_verify(s, case, g, dev, normal):
    _, new = _ragged(dict(case, ctx=0))
    cu, V, B = _starts(new), case["V"], case["B"]
    N = cu[-1]

    def noise(n):  # its largest, added to logits, is a sample of their softmax
        return -torch.log(-torch.log(torch.rand((n, V), generator=g, device=dev).clamp(1e-10, 1 - 1e-7)))

    x = 2 * normal(N, V)
    x[:, ::997] += 7  # the few tokens that are likely
    x = x.to(_TYPES[case["type"]])
    i = torch.cat([torch.arange(n) for n in new]).to(dev)
    parents = _tree(new, g, dev) if case["tree"] else None
    first = _ints(cu, dev).long()[:-1].repeat_interleave(_ints(new, dev).long())
    above = first + ((i - 1) if parents is None else parents.long()).clamp(min=0)
    # a drafting model that is about right: its logits are the target's and some noise
    tokens = torch.empty(N, dtype=torch.int32, device=dev)
    probs = torch.empty((N, V), device=dev) if case["probs"] else None
    for a in range(0, N, 256):
        row = x[above[a:a + 256]].float() + 0.5 * normal(len(above[a:a + 256]), V)
        tokens[a:a + 256] = (row + noise(len(row))).argmax(-1).int()
        if probs is not None:
            probs[a:a + 256] = torch.softmax(row, -1)
    temperature = None
    if case["temperature"] != 1.0:
        temperature = torch.full((B,), case["temperature"], device=dev)
        temperature[1::3] = 1.0
    s.update(x=x, tokens=tokens, cu=_ints(cu, dev), N=N, T=max(new), parents=parents, probs=probs,
             temperature=temperature, u=torch.rand(N, generator=g, device=dev))
    return s


def _request_of(s, rows, starts):
    t = torch.arange(rows, device=starts.device, dtype=torch.int32)
    b = torch.searchsorted(starts, t, right=True) - 1
    return b, t - starts[b]


def _gather(s, which, page, row):
    """Keys or values [.., hkv, D] in 32 bits at (page, row)."""
    c = s[which][page, row].float()
    if s[which].dtype != torch.int8:
        return c
    return c * s[which + "s"].transpose(1, 2)[page, row // _GROUP][..., None]


def _plain_attention(s):
    c = s["case"]
    B, T, hq, hkv, D, bs, L = c["B"], s["T"], c["hq"], c["hkv"], c["D"], c["block"], s["L"]
    dev = s["q"].device
    key = torch.arange(L, device=dev, dtype=torch.int32)
    page = s["table"][:, (key // bs).long()].long()
    row = (key % bs).long()[None].expand(B, L)
    k, v = (_gather(s, n, page, row).permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    b, i = _request_of(s, s["N"], s["cu"])
    i = i.long()
    q = torch.zeros((B, T, hq, D), device=dev)
    q[b, i] = s["q"]
    q = q.view(B, T, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, D)
    sc = (q @ k.transpose(2, 3).contiguous()) * (D ** -0.5)
    length = s["lengths"][b][:, None]
    j = key[None] - length  # a key's number among the request's new tokens
    if s["masks"] is None:
        see, at, depth = j <= i[:, None], key[None], i[:, None]
    else:
        bits = (s["masks"][:, None] >> torch.arange(64, device=dev)) & 1
        depths = torch.zeros((B, 64), dtype=torch.int64, device=dev)
        depths[b, i] = bits.sum(-1) - 1
        see = (j < 0) | ((j < 64) & (bits.gather(1, j.clamp(0, 63).long()) == 1))
        at = torch.where(j < 0, key[None], length + depths[b].gather(1, j.clamp(0, 63).long()))
        depth = bits.sum(-1, keepdim=True) - 1
    if c["window"]:
        see = see & ((length + depth - at < c["window"]) | (at < c["sinks"]))
    seen = torch.zeros((B, T, L), dtype=torch.bool, device=dev)
    seen[b, i] = see
    sc = sc.view(B, hkv, T, -1, L).masked_fill(~seen[:, None, :, None], -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38)).view(B, hkv, -1, L)
    n = e.sum(-1, keepdim=True)
    v = v.masked_fill((key[None] >= (s["starts"][1:] - s["starts"][:-1])[:, None])[:, None, :, None], 0.0)
    o = (e @ v) / torch.where(n == 0, torch.ones_like(n), n)
    return o.view(B, hkv, T, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(B, T, hq, D)[b, i]


def _store8(codes, scales, slots, y, need):
    """Values y [M, hkv, D], whose scales have to be `need` [M, hkv], to slots [M]: a
    group's scale is the largest needed by its new tokens and, where tokens lie
    before them, its own; those are rounded again by the new one."""
    nb, bs, hkv, D = codes.shape
    group, row = (slots // _GROUP).long(), slots % _GROUP
    n = nb * (bs // _GROUP)
    most = torch.zeros((n, hkv), device=y.device).index_reduce_(0, group, need, "amax")
    first = torch.full((n,), _GROUP, dtype=torch.int32, device=y.device).index_reduce_(0, group, row, "amin")
    old = scales.transpose(1, 2).reshape(n, hkv)
    held = ((first > 0) & (first < _GROUP))[:, None]
    fresh = torch.where((first < _GROUP)[:, None], torch.maximum(most, torch.where(held, old, 0 * old)), old)
    inverse = torch.where(fresh >= 2.0 ** -126, 1 / fresh, 0 * fresh)
    c = codes.reshape(n, _GROUP, hkv, D)
    again = torch.round(c.float() * (old * inverse)[:, None, :, None]).clamp(-127, 127).to(torch.int8)
    before = torch.arange(_GROUP, device=y.device)[None] < first[:, None]
    c = torch.where((held & (fresh > old))[:, None, :, None] & before[:, :, None, None], again, c)
    c[group, row.long()] = torch.round(y * inverse[group][..., None]).clamp(-127, 127).to(torch.int8)
    codes.copy_(c.view(nb, bs, hkv, D))
    scales.copy_(fresh.view(nb, bs // _GROUP, hkv).transpose(1, 2))


def _plain_read(s, first, starts, rows):
    b, i = _request_of(s, rows, starts)
    number = i if first is None else first[b] + i
    bs = s["case"]["block"]
    page = s["table"][b, (number // bs).long()].long()
    row = (number % bs).long()
    return tuple(_gather(s, w, page, row).half() for w in ("k", "v"))


def _plain_write(s):
    c = s["case"]
    N, hq, hkv, D, rot = s["N"], c["hq"], c["hkv"], c["D"], c["rot"]
    x = s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]
    q, k, v = (x[:, a * D:b * D].reshape(N, -1, D)
               for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    if s["qw"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["qw"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["kw"]
    cs = s["rope"][s["positions"].long()][:, None]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]

    def turn(h):
        if c["interleaved"]:
            a, b = h[..., 0:rot:2], h[..., 1:rot:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = h[..., :rot // 2], h[..., rot // 2:rot]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, h[..., rot:]], -1)

    k = turn(k)
    _store8(s["k"], s["ks"], s["slots"], k, k.abs().amax(-1) / 127)
    _store8(s["v"], s["vs"], s["slots"], v, v.abs().amax(-1) / 127)
    k, v = _plain_read(s, None, s["starts"], s["held"])
    return dict(q=turn(q), k=k, v=v)


def _plain_keep(s):
    c = s["case"]
    N, bs = s["N"], c["block"]
    b, d = _request_of(s, N, s["cu"])
    moved = (d < s["accepted"][b]) & (s["path"] != d)
    here, there = s["lengths"][b] + d, s["lengths"][b] + torch.where(moved, s["path"], d)
    page, at = s["table"][b, (there // bs).long()].long(), (there % bs).long()
    slot = s["table"][b, (here // bs).long()] * bs + here % bs
    if c["cache"] != "i8":
        k, v = s["k"][page, at], s["v"][page, at]
        s["k"][(slot // bs).long(), (slot % bs).long()] = k
        s["v"][(slot // bs).long(), (slot % bs).long()] = v
        return dict(k=s["k"], v=s["v"])
    parts = []
    for w in ("k", "v"):
        code = s[w][page, at].float()
        scale = s[w + "s"].transpose(1, 2)[page, at // _GROUP]
        parts.append((s[w], s[w + "s"], slot[moved], (code * scale[..., None])[moved],
                      (scale * (code.abs().amax(-1) / 127))[moved]))
    for p in parts:
        _store8(*p)
    k, v = _plain_read(s, s["lengths"], s["cu"], N)
    return dict(k=k, v=v)


def _plain_verify(s):
    c = s["case"]
    B, T, V, N = c["B"], s["T"], c["V"], s["N"]
    dev = s["x"].device
    b, i = _request_of(s, N, s["cu"])
    i = i.long()
    new = (s["cu"][1:] - s["cu"][:-1]).long()
    first = s["cu"].long()[b]
    x = s["x"].double()
    temp = torch.ones(B, device=dev) if s["temperature"] is None else s["temperature"]
    z = (x - x.amax(-1, keepdim=True)) / torch.where(temp > 0, temp, torch.ones_like(temp)).double()[b][:, None]
    e = torch.exp(z)
    p = e / e.sum(-1, keepdim=True)
    if s["temperature"] is not None:
        top = (x == x.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True)  # the first of equal ones
        best = torch.zeros_like(p).scatter_(1, top, 1.0)
        p = torch.where((temp > 0)[b][:, None], p, best)
    up = (i - 1) if s["parents"] is None else s["parents"].long()
    of = p[first + up.clamp(min=0)].gather(1, s["tokens"].long()[:, None])[:, 0]  # of each token
    # tokens of one request against each other, [B, T, T]
    here = torch.zeros((B, T), dtype=torch.bool, device=dev)
    here[b, i] = True

    def pad(v, fill):
        r = torch.full((B, T), fill, dtype=v.dtype, device=dev)
        r[b, i] = v
        return r

    par, tok, prob, u = pad(up, -9), pad(s["tokens"].long(), -1), pad(of, 0.0), pad(s["u"].double(), 0.0)
    earlier = torch.ones((T, T), dtype=torch.bool, device=dev).tril(-1)
    sibling = (par[:, :, None] == par[:, None, :]) & earlier & here[:, None, :]
    again = (sibling & (tok[:, :, None] == tok[:, None, :])).any(-1)  # refused before already
    prob = torch.where(again, 0 * prob, prob)
    if s["probs"] is None:
        mass = 1 - (sibling * prob[:, None, :]).sum(-1)
        good = u * mass < prob
    else:
        q = pad(s["probs"].gather(1, s["tokens"].long()[:, None])[:, 0].double(), 1.0)
        good = u * q < prob
    good = good & here & (par >= 0)
    good = good & ~(sibling & good[:, None, :]).any(-1)
    good[:, 0] = new > 0
    # accepted: the token and all that it descends from
    up_to = torch.eye(T, dtype=torch.float64, device=dev).repeat(B, 1, 1)
    up_to.scatter_(2, par.clamp(min=0)[:, :, None], 1.0)

    def twice(m):
        return (m @ m).clamp(max=1.0)

    up_to = twice(twice(twice(twice(twice(twice(up_to))))))  # depths below 64
    kept = good & ((up_to * (~good[:, None, :])).sum(-1) == 0)
    accepted = kept.sum(-1)
    rank = kept.cumsum(-1) - 1
    path = torch.full((B, T + 1), -1, dtype=torch.int64, device=dev)
    path.scatter_(1, torch.where(kept, rank, T), torch.arange(T, device=dev).repeat(B, 1))
    last = path.gather(1, (accepted - 1).clamp(min=0)[:, None])[:, 0]
    row = s["cu"].long()[:-1] + last
    r = p[row]
    child = (par == last[:, None]) & here
    if s["probs"] is None:
        refused = torch.zeros((B, V), device=dev).index_put_(
            (torch.arange(B, device=dev)[:, None].expand(B, T)[child], tok[child]), torch.ones((), device=dev))
        left = torch.where(refused > 0, 0 * r, r)
    else:
        drafted = s["probs"][(row + 1).clamp(max=N - 1)].double()
        left = torch.where((child.sum(-1) > 0)[:, None], (r - drafted).clamp(min=0), r)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, r)
    total = left.cumsum(-1)
    at = s["u"][s["cu"].long()[:-1]].double()[:, None] * total[:, -1:]
    return dict(accepted=accepted.int(), path=path[b, i].int(), next_tokens=(total <= at).sum(-1).int())


def run(state):
    s = state
    if not own:
        return {"attention": _plain_attention, "window": _plain_attention, "write": _plain_write,
                "verify": _plain_verify, "keep": _plain_keep}[s["op"]](s)
    from forge_amd import step
    c = s["case"]
    if s["op"] == "verify":
        r = step.verify_draft(s["x"], s["tokens"], s["cu"], s["u"], parents=s["parents"],
                              draft_probs=s["probs"], temperature=s["temperature"])
        return dict(accepted=r.accepted, path=r.path, next_tokens=r.next_tokens)
    k, v = s["k"], s["v"]
    if k.dtype == torch.int8:
        k, v = step.Cache8(k, s["ks"]), step.Cache8(v, s["vs"])
    if s["op"] in ("attention", "window"):
        return step.tree_attention(s["q"], k, v, s["table"], s["lengths"], s["cu"], masks=s["masks"],
                                   max_new=s["T"], window=c["window"] or None, sinks=c["sinks"])
    if s["op"] == "write":
        q = step.qk_norm_rope(s["qkv"], s["positions"], s["slots"], s["rope"], k, v, bias=s["bias"],
                              q_weight=s["qw"], k_weight=s["kw"], eps=1e-6, interleaved=c["interleaved"])
        k, v = step.read_cache(k, v, s["table"], s["starts"], s["held"])
        return dict(q=q, k=k, v=v)
    step.keep_accepted(k, v, s["table"], s["lengths"], s["cu"], s["path"], s["accepted"])
    if c["cache"] == "i8":
        k, v = step.read_cache(k, v, s["table"], s["cu"], s["N"], first=s["lengths"])
    return dict(k=k, v=v)


def _values64(s, which):
    x = s[which].double()
    if s[which].dtype == torch.int8:
        nb, bs, hkv, D = x.shape
        x = x.view(nb, bs // _GROUP, _GROUP, hkv, D) * s[which + "s"].double().transpose(1, 2)[:, :, None, :, None]
        x = x.view(nb, bs, hkv, D)
    return x


def _exact_attention(s):
    c = s["case"]
    ctx, new = _ragged(c)
    bs, hq, hkv, D = c["block"], c["hq"], c["hkv"], c["D"]
    out, at = [], 0
    for b in range(c["B"]):
        n, L = new[b], ctx[b] + new[b]
        pages = s["table"][b, :-(-L // bs)].long()
        part = {w: s[w].index_select(0, pages) for w in ("k", "v")}
        if s["k"].dtype == torch.int8:
            part.update({w: s[w].index_select(0, pages) for w in ("ks", "vs")})
        k, v = (_values64(part, w).flatten(0, 1)[:L].transpose(0, 1).contiguous() for w in ("k", "v"))
        q = s["q"][at:at + n].double().view(n, hkv, hq // hkv, D).transpose(0, 1).reshape(hkv, -1, D)
        sc = torch.bmm(q, k.transpose(1, 2).contiguous()).view(hkv, n, -1, L) / math.sqrt(D)
        draft = torch.ones((n, n), dtype=torch.bool, device=q.device).tril()
        if s["masks"] is not None:
            draft = (s["masks"][at:at + n, None] >> torch.arange(n, device=q.device)) & 1 == 1
        see = torch.cat([torch.ones((n, ctx[b]), dtype=torch.bool, device=q.device), draft], 1)
        if c["window"]:
            place = torch.arange(L, device=q.device)
            place[ctx[b]:] = ctx[b] + draft.sum(-1) - 1
            apart = place[ctx[b]:, None] - place[None]
            see &= (apart < c["window"]) | (place < c["sinks"])[None]
        sc.masked_fill_(~see[None, :, None], -math.inf)
        p = torch.softmax(sc, -1).reshape(hkv, -1, L)
        out.append(torch.bmm(p, v).view(hkv, n, -1, D).transpose(0, 1).reshape(n, hq, D))
        at += n
    return torch.cat(out)


def _quantised64(held, scales, rows, amax):
    """A group's values after rows [m, hkv, D] came behind held ones [h, hkv, D] (codes), and its scales."""
    old = scales if len(held) else torch.zeros_like(scales)
    new = torch.maximum(old, amax.amax(0) / 127)
    step = torch.where(new > 0, new, torch.ones_like(new))[None, :, None]
    again = torch.where((new > old)[None, :, None], torch.round(held * (old[None, :, None] / step)), held)
    return torch.cat([again, torch.round(rows / step).clamp(-127, 127)]) * new[None, :, None], new


def _exact_rows(s, which, rows, amax, first, counts):
    """The requests' tokens in 64 bits once rows are written, counts[b] of request b from its
    number first[b] on."""
    c, out, at = s["case"], [], 0
    bs = c["block"]
    for b in range(c["B"]):
        end, parts = first[b] + counts[b], []
        pages = s["table"][b].tolist()
        for g0 in range(0, max(end, 1), _GROUP):
            page, r = pages[g0 // bs], g0 % bs
            codes, scale = s[which][page, r:r + _GROUP].double(), s[which + "s"][page, :, r // _GROUP].double()
            if g0 + _GROUP <= first[b] or counts[b] == 0:
                parts.append((codes * scale[None, :, None])[:end - g0])
                continue
            h, m = max(0, first[b] - g0), min(end, g0 + _GROUP) - max(g0, first[b])
            parts.append(_quantised64(codes[:h], scale, rows[at:at + m], amax[at:at + m])[0])
            at += m
        out.append(torch.cat(parts)[:end])
    return out


def _exact_write(s):
    c = s["case"]
    ctx, new = _ragged(c)
    N, hq, hkv, D, rot = s["N"], c["hq"], c["hkv"], c["D"], c["rot"]
    x = s["qkv"].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x.view(N, hq + 2 * hkv, D)
    cs = s["rope"].double()[s["positions"].long()].view(N, 1, 2, rot // 2)
    z = torch.complex(cs[:, :, 0], cs[:, :, 1])
    heads = x[:, :hq + hkv]
    if s["qw"] is not None:
        w = torch.cat([s["qw"].double().expand(hq, D), s["kw"].double().expand(hkv, D)])
        heads = heads / ((heads ** 2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w
    part = heads[..., :rot]
    if c["interleaved"]:
        r = torch.view_as_real(torch.view_as_complex(part.reshape(N, -1, rot // 2, 2).contiguous())
                               * z).flatten(-2)
    else:
        r = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * z
        r = torch.cat([r.real, r.imag], -1)
    heads = torch.cat([r, heads[..., rot:]], -1)
    out = dict(q=heads[:, :hq])
    for w, rows in (("k", heads[:, hq:]), ("v", x[:, hq + hkv:])):
        out[w] = torch.cat(_exact_rows(s, w, rows, rows.abs().amax(-1), ctx, new))
    return out


def _exact_keep(s):
    c = s["case"]
    ctx, new = _ragged(c)
    bs = c["block"]
    path, accepted, at = s["path"].tolist(), s["accepted"].tolist(), 0
    values = {w: _values64(s, w) for w in ("k", "v")}
    result = {w: v.clone() for w, v in values.items()}
    out = {"k": [], "v": []}
    for b in range(c["B"]):
        pages = s["table"][b].tolist()
        kept = path[at:at + accepted[b]]
        moves = [(ctx[b] + p, ctx[b] + d) for d, p in enumerate(kept) if p != d]
        for w in ("k", "v"):
            if c["cache"] != "i8":
                for a, z in moves:
                    result[w][pages[z // bs], z % bs] = values[w][pages[a // bs], a % bs]
                continue
            for g in sorted({z // _GROUP for _, z in moves}):
                mine = [(a, z) for a, z in moves if z // _GROUP == g]
                page, r = pages[_GROUP * g // bs], _GROUP * g % bs
                rows = torch.stack([values[w][pages[a // bs], a % bs] for a, _ in mine])
                h = mine[0][1] - _GROUP * g
                codes, scale = s[w][page, r:r + _GROUP].double(), s[w + "s"][page, :, r // _GROUP].double()
                got, fresh = _quantised64(codes[:h], scale, rows, rows.abs().amax(-1))
                # what lies behind is nobody's: its codes under the new scale
                result[w][page, r:r + _GROUP] = torch.cat([got, codes[len(got):] * fresh[None, :, None]])
            out[w] += [result[w][pages[n // bs], n % bs] for n in range(ctx[b], ctx[b] + new[b])]
        at += new[b]
    return result if c["cache"] != "i8" else {w: torch.stack(v) for w, v in out.items()}


def exact(case, seed):
    """The operators' definitions in 64 bits; what is verified are whole numbers."""
    if case["op"] == "verify":
        return None
    s = prepare(case, seed)
    return {"attention": _exact_attention, "window": _exact_attention, "write": _exact_write,
            "keep": _exact_keep}[case["op"]](s)


def work(case):
    op = case["op"]
    if op == "verify":
        new = _ragged(dict(case, ctx=0))[1]
        N, V, size = sum(new), case["V"], 4 if case["type"] == "f32" else 2
        # the logits, one row of draft probabilities a request; a token's own in and out
        return {"bytes": N * (size * V + 20) + 12 * case["B"] + 4 * case["B"] * V * case["probs"],
                "flops": 4 * N * V}
    ctx, new = _ragged(case)
    hkv, D = case["hkv"], case["D"]
    if op == "write":
        N, hq = sum(new), case["hq"]
        read = 4 * (hq + 2 * hkv) * D + 4 * case["rot"] + 8
        held = N + sum(ctx)
        # the step's rows in, queries and codes out; all codes in, values in 16 bits out
        return {"bytes": N * (read + 4 * hq * D + 2 * hkv * D) + held * 2 * hkv * D * (1 + 2),
                "flops": N * (hq + hkv) * 3 * case["rot"] + 4 * N * hkv * D}
    if op == "keep":
        size = 1 if case["cache"] == "i8" else 2
        moved = sum(0.3 * n for n in new)
        back = sum(new) * 2 * hkv * D * 3 if case["cache"] == "i8" else 0
        return {"bytes": int(moved * 4 * hkv * D * size + back + 4 * sum(new) + 16 * case["B"]), "flops": 0}
    hq = case["hq"]
    keys = [c + n for c, n in zip(ctx, new)]
    if case["window"]:
        keys = [min(k, n + case["window"] + case["sinks"]) for k, n in zip(keys, new)]
    size = 2 * (D + 4 / _GROUP) if case["cache"] == "i8" else 4 * D
    return {"bytes": int(sum(keys) * hkv * size) + 8 * sum(new) * hq * D,
            "flops": sum(4 * n * hq * D * k for n, k in zip(new, keys))}
