"""The operators of a decoding or verifying step that surround the quantized
matmuls, measured through forge_amd.step.

A case is one operator of a serving step over a paged cache:

  plan       plan_step: cache blocks, slots, positions and tree masks of the
             step's tokens, from the requests' lengths
  rope       qk_norm_rope: bias, per-head norm and rotation of fused_qkv's rows,
             keys and values written to their cache slots
  attention  tree_attention: each request's drafted tokens over its cached
             context and over the tokens of the draft that they descend from
  logprobs   token_logprobs: log probabilities of given tokens over the head's
             rows, the entropy and the most likely alternatives

Heads: 32 query and 4 key heads of 64 (a small model, hidden 2048), 28 and 4 of
128 (7B, hidden 3584), 32 and 8 of 128 (8B, hidden 4096), and generic ones.
`own` false computes the operators from elementary torch operations in 32 bits;
`own` true calls forge_amd.step.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_ROPE_TABLE = 32768  # positions of the rotation table that a program keeps


def listed():
    return [
        # one request of a small model, a short chain of drafted tokens: latency
        dict(name="attention, one short chain", op="attention", B=1, ctx=333, T=4, tree=False,
             hq=32, hkv=4, D=64, block=16, cache="f16"),
        # a batch that decodes one token each, 7B heads (7 query heads a key head)
        dict(name="attention, decode batch", op="attention", B=48, ctx=2001, T=1, tree=False,
             hq=28, hkv=4, D=128, block=16, cache="bf16"),
        # eight requests that verify a drafted tree, 8B heads
        dict(name="attention, trees of 8", op="attention", B=8, ctx=4097, T=25, tree=True,
             hq=32, hkv=8, D=128, block=16, cache="f16"),
        # one long document: the context is split over the whole card
        dict(name="attention, long context", op="attention", B=1, ctx=131000, T=13, tree=True,
             hq=28, hkv=4, D=128, block=64, cache="bf16"),
        # a full batch of large trees: the largest attention call
        dict(name="attention, full batch", op="attention", B=32, ctx=8190, T=32, tree=True,
             hq=32, hkv=8, D=128, block=32, cache="f16"),
        # one decoded token of a small model through its rotation: latency
        dict(name="rope, one token", op="rope", N=1, hq=32, hkv=4, D=64, rot=64, block=16,
             cache="f16", bias=False, norm=False, interleaved=True),
        # a verified batch of a 7B model, whose projections have a bias
        dict(name="rope, verified batch", op="rope", N=203, hq=28, hkv=4, D=128, rot=128, block=16,
             cache="bf16", bias=True, norm=False, interleaved=False),
        # a long prompt with normalized heads: bandwidth
        dict(name="rope, prompt", op="rope", N=4095, hq=32, hkv=8, D=128, rot=128, block=32,
             cache="f16", bias=False, norm=True, interleaved=False),
        # the logits of one verified chain, five alternatives each
        dict(name="logprobs, one chain", op="logprobs", M=5, V=32000, top=5, J=1, type="f32",
             masked=False),
        # the logits of a verified batch over the largest vocabulary
        dict(name="logprobs, full batch", op="logprobs", M=501, V=152064, top=20, J=2, type="f32",
             masked=False),
        # a few requests with drafted trees
        dict(name="plan, few trees", op="plan", B=7, ctx=1500, T=25, tree=True, block=16),
        # a large batch with a chunk of prompt each
        dict(name="plan, large batch", op="plan", B=1500, ctx=4000, T=130, tree=False, block=32),
    ]


_HEADS = [(32, 4, 64), (28, 4, 128), (32, 8, 128), (12, 12, 64), (9, 3, 96), (10, 2, 256), (5, 1, 128)]


def _log(rng, lo, hi):
    n = min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))
    return n - 1 if n == 3072 else n


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, no
    larger than the largest listed case of its operator."""
    op = rng.choice(["attention", "attention", "rope", "logprobs", "plan"])
    block = rng.choice([16, 32, 64, 128])
    hq, hkv, D = rng.choice(_HEADS)
    if op == "attention":
        tree = rng.random() < 0.6
        B, T = _log(rng, 1, 64), _log(rng, 1, 64)
        most = min(131072, 32 * 8190 * 8 * 128 // (B * hkv * D), 32 * 32 * 32 * 8190 // (B * T * hq))
        return dict(op=op, B=B, ctx=_log(rng, 1, max(1, most)), T=T, tree=tree, hq=hq, hkv=hkv, D=D,
                    block=block, cache=rng.choice(["f16", "bf16"]))
    if op == "rope":
        most = 4095 * 48 * 128 // ((hq + 2 * hkv) * D)
        return dict(op=op, N=_log(rng, 1, most), hq=hq, hkv=hkv, D=D,
                    rot=rng.choice([D, D, D // 2]), block=block, cache=rng.choice(["f16", "bf16"]),
                    bias=rng.random() < 0.3, norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.3)
    if op == "logprobs":
        V = _log(rng, 1000, 200000)
        return dict(op=op, M=_log(rng, 1, 501 * 152064 // V if V > 50000 else 1500), V=V,
                    top=rng.randrange(0, 33), J=rng.choice([1, 1, 1, 3]),
                    type=rng.choice(["f32", "f32", "f16", "bf16"]), masked=rng.random() < 0.3)
    tree = rng.random() < 0.5
    return dict(op=op, B=_log(rng, 1, 1500), ctx=_log(rng, 1, 4000),
                T=_log(rng, 1, 64 if tree else 130), tree=tree, block=block)


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
    """Parents [N] of random trees: of a request's tokens the first ones hang on
    the context, token i on one of the tokens before it, or on the context."""
    i = torch.cat([torch.arange(n) for n in new]).to(dev)
    r = torch.rand(i.shape, generator=g, device=dev)
    return (torch.floor(r.sqrt() * (i + 1)).to(torch.int32) - 1).clamp(max=i.to(torch.int32) - 1)


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


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    op = case["op"]
    s = dict(op=op, case=case)
    if op in ("attention", "plan"):
        ctx, new = _ragged(case)
        cu, bs = _starts(new), case["block"]
        s.update(N=cu[-1], T=max(new), L=max(c + n for c, n in zip(ctx, new)),
                 lengths=_ints(ctx, dev), new=_ints(new, dev))
        held = [-(-(c + n if op == "attention" else c) // bs) for c, n in zip(ctx, new)]
        wide = max(-(-(c + n) // bs) for c, n in zip(ctx, new))
        spare = sum(-(-(c + n) // bs) for c, n in zip(ctx, new)) - sum(held)
        n = sum(held) + spare + (1000 if op == "plan" else 0)  # a plan's pool has more
        blocks = torch.randperm(n, generator=g, device=dev).to(torch.int32)
        table = torch.zeros((case["B"], wide), dtype=torch.int32, device=dev)
        have = torch.arange(wide, device=dev)[None] < _ints(held, dev)[:, None]
        table[have] = blocks[:sum(held)]
        s["table"] = table
        if op == "plan":
            s.update(free=blocks[sum(held):].contiguous(),
                     parents=_tree(new, g, dev) if case["tree"] else None)
            return s
        hq, hkv, D = case["hq"], case["hkv"], case["D"]
        # a block's rows lie head by head, as paged_cache() lays them out
        s["k"], s["v"] = (normal(n, hkv, bs, D).to(_TYPES[case["cache"]]).transpose(1, 2)
                          for _ in range(2))
        s.update(q=2 * normal(cu[-1], hq, D), cu=_ints(cu, dev),
                 masks=_masks64(_tree(new, g, dev), new) if case["tree"] else None)
        return s
    if op == "rope":
        N, hq, hkv, D, rot = (case[k] for k in ("N", "hq", "hkv", "D", "rot"))
        rows = (hq + 2 * hkv) * D
        n = -(-2 * N // case["block"])
        x = normal(N, rows)
        x[:, ::61] *= 6  # a few strong channels, as projections have them
        angle = torch.arange(_ROPE_TABLE, device=dev, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        k, v = (torch.zeros((n, hkv, case["block"], D), dtype=_TYPES[case["cache"]],
                            device=dev).transpose(1, 2) for _ in range(2))
        s.update(qkv=x, k=k, v=v, table=torch.cat([angle.cos(), angle.sin()], 1).float(),
                 positions=torch.randint(0, _ROPE_TABLE, (N,), generator=g, device=dev).int(),
                 slots=torch.randperm(n * case["block"], generator=g, device=dev)[:N].int(),
                 bias=normal(rows) if case["bias"] else None,
                 qw=1 + 0.2 * normal(D) if case["norm"] else None,
                 kw=1 + 0.2 * normal(D) if case["norm"] else None)
        return s
    M, V = case["M"], case["V"]
    x = 2.5 * normal(M, V)
    x[:, ::997] += 6  # the few tokens that are likely
    if case["masked"]:
        x[torch.rand((M, V), generator=g, device=dev) < 0.3] = -math.inf
        x[:, ::31] = 0.0  # some tokens are always allowed
    s.update(x=x.to(_TYPES[case["type"]]),
             targets=torch.randint(0, (V - 1) // 31 + 1, (M, case["J"]), generator=g,
                                   device=dev).int() * 31)
    return s


def _plain_plan(s):
    bs, table, N = s["case"]["block"], s["table"], s["N"]
    dev = table.device
    have = (s["lengths"] + bs - 1) // bs
    want = (s["lengths"] + s["new"] + bs - 1) // bs
    cu = torch.cat([s["new"].new_zeros(1), s["new"].cumsum(0, dtype=torch.int32)])
    taken = (want - have).cumsum(0, dtype=torch.int32)
    col = torch.arange(table.shape[1], device=dev, dtype=torch.int32)[None]
    place = (taken - (want - have))[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    free = s["free"] if s["free"].numel() else s["free"].new_zeros(1)
    table.copy_(torch.where(fresh, free[place.clamp(0, free.numel() - 1).long()], table))
    t = torch.arange(N, device=dev, dtype=torch.int32)
    b = torch.searchsorted(cu, t, right=True) - 1
    i = t - cu[b]
    at = s["lengths"][b] + i
    slots = table[b, (at // bs).long()] * bs + at % bs
    masks = depth = None
    if s["parents"] is not None:
        up = torch.zeros((len(cu) - 1, 64, 65), device=dev)
        up[b, i.long(), (s["parents"].long() + 65) % 65] = 1.0  # the context, -1: column 64
        up[b, i.long(), i.long()] = 1.0
        up = up[:, :, :64]

        def twice(m):
            return (m @ m).clamp(max=1.0)

        up = twice(twice(twice(twice(twice(twice(up))))))[b, i.long()].long()
        depth = up.sum(-1, dtype=torch.int32) - 1
        masks = (up << torch.arange(64, device=dev)).sum(-1)
    positions = s["lengths"][b] + (i if depth is None else depth)
    return dict(cu=cu, slots=slots, positions=positions, masks=masks, table=table,
                info=torch.stack([taken[-1], torch.zeros_like(taken[-1])]))


def _plain_rope(s):
    c = s["case"]
    N, hq, hkv, D, rot = (c[k] for k in ("N", "hq", "hkv", "D", "rot"))
    x = s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]
    q, k, v = (x[:, a * D:b * D].reshape(N, -1, D)
               for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv)))
    if s["qw"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["qw"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["kw"]
    cs = s["table"][s["positions"].long()][:, None]
    cos, sin = cs[..., :rot // 2], cs[..., rot // 2:]

    def turn(h):
        if c["interleaved"]:
            a, b = h[..., 0:rot:2], h[..., 1:rot:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = h[..., :rot // 2], h[..., rot // 2:rot]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([r, h[..., rot:]], -1)

    slots = s["slots"].long()
    at = (slots // c["block"], slots % c["block"])
    s["k"][at] = turn(k).to(s["k"].dtype)
    s["v"][at] = v.to(s["v"].dtype)
    return dict(q=turn(q), k=s["k"], v=s["v"])


def _plain_attention(s):
    c = s["case"]
    B, T, hq, hkv, D, bs, L = c["B"], s["T"], c["hq"], c["hkv"], c["D"], c["block"], s["L"]
    dev = s["q"].device
    key = torch.arange(L, device=dev, dtype=torch.int32)
    page = s["table"][:, (key // bs).long()].long()
    row = (key % bs).long()[None].expand(B, L)
    k, v = (s[n][page, row].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    t = torch.arange(s["N"], device=dev, dtype=torch.int32)
    b = torch.searchsorted(s["cu"], t, right=True) - 1
    i = (t - s["cu"][b]).long()
    q = torch.zeros((B, T, hq, D), device=dev)
    q[b, i] = s["q"]
    q = q.view(B, T, hkv, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, D)
    sc = (q @ k.transpose(2, 3).contiguous()) * (D ** -0.5)
    seen = torch.zeros((B, T, L), dtype=torch.bool, device=dev)
    j = key[None] - s["lengths"][b][:, None]  # a key's number among the request's new tokens
    if s["masks"] is None:
        seen[b, i] = j <= i[:, None]
    else:
        bits = (s["masks"][:, None] >> j.clamp(0, 63)) & 1
        seen[b, i] = (j < 0) | ((j < 64) & (bits == 1))
    sc = sc.view(B, hkv, T, -1, L).masked_fill(~seen[:, None, :, None], -math.inf)
    e = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38)).view(B, hkv, -1, L)
    n = e.sum(-1, keepdim=True)
    v = v.masked_fill((key[None] >= (s["lengths"] + s["new"])[:, None])[:, None, :, None], 0.0)
    o = (e @ v) / torch.where(n == 0, torch.ones_like(n), n)
    return o.view(B, hkv, T, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(B, T, hq, D)[b, i]


def _plain_logprobs(s):
    x, top = s["x"].float(), s["case"]["top"]
    V = x.shape[1]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    n = e.sum(-1, keepdim=True)
    lse = m + torch.log(n)
    seen = torch.where(e > 0, (x - m) * e, torch.zeros_like(e)).sum(-1, keepdim=True)
    out = dict(logprobs=x.gather(1, s["targets"].long()) - lse,
               entropy=(torch.log(n) - seen / n)[:, 0])
    if top:
        # an integer in the order of the value, and of the token where values tie
        w = (x + 0.0).view(torch.int32)
        w = torch.where(w < 0, w ^ 0x7FFFFFFF, w).long() * (1 << 32)
        best = (w + torch.arange(V - 1, -1, -1, device=x.device)).topk(top, -1).values
        token = V - 1 - (best & 0xFFFFFFFF)
        out.update(top_logprobs=x.gather(1, token) - lse, top_tokens=token.int())
    return out


def run(state):
    s = state
    if not own:
        return {"plan": _plain_plan, "rope": _plain_rope, "attention": _plain_attention,
                "logprobs": _plain_logprobs}[s["op"]](s)
    from forge_amd import step
    c = s["case"]
    if s["op"] == "plan":
        p = step.plan_step(s["lengths"], s["new"], s["table"], s["free"], c["block"], s["N"],
                           parents=s["parents"])
        return dict(cu=p.cu, slots=p.slots, positions=p.positions, masks=p.masks, table=s["table"],
                    info=p.info)
    if s["op"] == "rope":
        q = step.qk_norm_rope(s["qkv"], s["positions"], s["slots"], s["table"], s["k"], s["v"],
                              bias=s["bias"], q_weight=s["qw"], k_weight=s["kw"], eps=1e-6,
                              interleaved=c["interleaved"])
        return dict(q=q, k=s["k"], v=s["v"])
    if s["op"] == "attention":
        return step.tree_attention(s["q"], s["k"], s["v"], s["table"], s["lengths"], s["cu"],
                                   masks=s["masks"], max_new=s["T"])
    r = step.token_logprobs(s["x"], s["targets"], top=c["top"])
    out = dict(logprobs=r.logprobs, entropy=r.entropy)
    if c["top"]:
        out.update(top_logprobs=r.top_logprobs, top_tokens=r.top_tokens)
    return out


def _exact_attention(s):
    c = s["case"]
    ctx, new = _ragged(c)
    bs, hq, hkv, D = c["block"], c["hq"], c["hkv"], c["D"]
    out, at = [], 0
    for b in range(c["B"]):
        n, L = new[b], ctx[b] + new[b]
        pages = s["table"][b, :-(-L // bs)].long()
        k, v = (s[w].index_select(0, pages).flatten(0, 1)[:L].double().transpose(0, 1).contiguous()
                for w in ("k", "v"))  # [hkv, L, D]
        q = s["q"][at:at + n].double().view(n, hkv, hq // hkv, D).transpose(0, 1).reshape(hkv, -1, D)
        sc = torch.bmm(q, k.transpose(1, 2).contiguous()).view(hkv, n, -1, L) / math.sqrt(D)
        draft = torch.ones((n, n), dtype=torch.bool, device=q.device).tril()
        if s["masks"] is not None:
            draft = (s["masks"][at:at + n, None] >> torch.arange(n, device=q.device)) & 1 == 1
        sc[..., ctx[b]:].masked_fill_(~draft[None, :, None], -math.inf)
        p = torch.softmax(sc, -1).reshape(hkv, -1, L)
        out.append(torch.bmm(p, v).view(hkv, n, -1, D).transpose(0, 1).reshape(n, hq, D))
        at += n
    return torch.cat(out)


def _exact_rope(s):
    c = s["case"]
    N, hq, hkv, D, rot = (c[k] for k in ("N", "hq", "hkv", "D", "rot"))
    x = s["qkv"].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()
    x = x.view(N, hq + 2 * hkv, D)
    cs = s["table"].double()[s["positions"].long()].view(N, 1, 2, rot // 2)
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
    k, v = (torch.zeros(s[w].shape, dtype=torch.float64, device=x.device) for w in ("k", "v"))
    for cache, rows in ((k, heads[:, hq:]), (v, x[:, hq + hkv:])):
        cache.view(-1, hkv, D)[s["slots"].long()] = rows
    return dict(q=heads[:, :hq], k=k, v=v)


def _exact_logprobs(s):
    out = dict(logprobs=[], entropy=[], top_logprobs=[])
    for x, t in zip(s["x"].split(64), s["targets"].split(64)):
        lp = torch.log_softmax(x.double(), -1)
        out["logprobs"].append(lp.gather(1, t.long()))
        out["entropy"].append(torch.special.entr(lp.exp()).sum(-1))
        if s["case"]["top"]:
            out["top_logprobs"].append(lp.topk(s["case"]["top"], -1).values)
    return {k: torch.cat(v) if v else None for k, v in out.items()}


def exact(case, seed):
    """The operators' definitions in 64 bits; a plan's outputs are whole numbers."""
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rope": _exact_rope, "logprobs": _exact_logprobs}[case["op"]](s)


def work(case):
    op = case["op"]
    if op == "plan":
        ctx, new = _ragged(case)
        N, B, bs = sum(new), case["B"], case["block"]
        fresh = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        # lengths, new tokens, parents, free blocks in; starts, table entries,
        # slots, positions and masks out
        return {"bytes": 12 * B + 8 * fresh + N * (8 + (12 if case["tree"] else 0)), "flops": 0}
    if op == "rope":
        N, hq, hkv, D = (case[k] for k in ("N", "hq", "hkv", "D"))
        read = 4 * (hq + 2 * hkv) * D + 4 * case["rot"] + 8
        return {"bytes": N * (read + 4 * hq * D + 2 * 2 * hkv * D),
                "flops": N * (hq + hkv) * (3 * case["rot"] + 4 * D * case["norm"])}
    if op == "logprobs":
        M, V, size = case["M"], case["V"], 4 if case["type"] == "f32" else 2
        return {"bytes": M * (size * V + 8 * case["J"] + 4 + 8 * case["top"]), "flops": 6 * M * V}
    ctx, new = _ragged(case)
    hq, hkv, D = case["hq"], case["hkv"], case["D"]
    keys = sum(c + n for c, n in zip(ctx, new))
    return {"bytes": 4 * keys * hkv * D + 8 * sum(new) * hq * D,
            "flops": sum(4 * n * hq * D * (c + n) for c, n in zip(ctx, new))}
