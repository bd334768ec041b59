"""Plain 64-bit implementations of the step operators for caches of 8 bits, windows and
drafts (include/forge_step.h), from their definitions, one request and group at a time."""
from __future__ import annotations

import numpy as np
import torch

GROUP = 16


def values(codes, scales):
    """A cache of 8 bits [blocks, block size, kv heads, D] in 64 bits."""
    s = scales.double()
    s = torch.where((s > 0) & (s < np.inf), s, torch.zeros_like(s))
    return codes.double() * s.transpose(1, 2).repeat_interleave(GROUP, 1)[..., None]


def sees(length, n, masks, window, sinks):
    """[n, length + n]: which keys a request's new tokens see."""
    keys = length + n
    see = torch.zeros((n, keys), dtype=torch.bool)
    see[:, :length] = True
    place = list(range(length)) + [0] * n
    draft = []
    for i in range(n):
        bits = {j for j in range(i + 1)} if masks is None else {j for j in range(min(n, 64)) if int(masks[i]) >> j & 1}
        draft.append(bits)
        place[length + i] = length + (i if masks is None else max(bin(int(masks[i]) % 2 ** 64).count("1") - 1, 0))
        for j in bits:
            see[i, length + j] = True
    if window:
        # (a new key's position, as the token that sees it counts it: how many bits of its mask lie below)
        for i in range(n):
            for j in range(keys):
                at = j if j < length else length + len([x for x in draft[i] if x < j - length])
                if not (place[length + i] - at < window or at < sinks):
                    see[i, j] = False
    return see


def attention(q, k, v, table, lengths, cu, masks, scale, window=0, sinks=0):
    """fp64 [N, hq, D] over 64-bit caches; keys that are not seen take no part."""
    N, hq, D = q.shape
    bs, hkv = k.shape[1:3]
    out = torch.zeros((N, hq, D), dtype=torch.float64)
    for b in range(len(lengths)):
        t0, n = int(cu[b]), int(cu[b + 1]) - int(cu[b])
        if n == 0:
            continue
        ln = int(lengths[b])
        keys = ln + n
        pages = table[b, :-(-keys // bs)].long()
        there = (pages >= 0) & (pages < len(k))
        at = pages.clamp(0, len(k) - 1)
        see = sees(ln, n, None if masks is None else masks[t0:t0 + n], window, sinks)
        see &= there.repeat_interleave(bs)[:keys][None]
        kk = torch.where(see.any(0)[:, None, None], k[at].flatten(0, 1)[:keys], 0.0).transpose(0, 1).contiguous()
        vv = torch.where(see.any(0)[:, None, None], v[at].flatten(0, 1)[:keys], 0.0).transpose(0, 1).contiguous()
        qq = q[t0:t0 + n].double().view(n, hkv, hq // hkv, D).permute(1, 0, 2, 3)  # [hkv, n, G, D]
        s = (qq.reshape(hkv, -1, D) @ kk.transpose(1, 2)).view(hkv, n, -1, keys) * scale
        s = s.masked_fill(~see[None, :, None], -np.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), 0.0) * see[None, :, None]
        o = (p.reshape(hkv, -1, keys) @ vv).view(hkv, n, -1, D)
        out[t0:t0 + n] = o.permute(1, 0, 2, 3).reshape(n, hq, D)
    return out


def enter(codes, scales, runs):
    """Groups after new tokens entered them.  codes [groups, 16, D], scales [groups] are changed;
    runs: (group, first row, values [m, D], needed scale) in 64 bits."""
    for g, first, x, need in runs:
        old = float(scales[g]) if first else 0.0
        s = max(need, old)
        inverse = 1 / s if s >= 2.0 ** -126 else 0.0
        if s > old:
            codes[g, :first] = np.rint(codes[g, :first] * (old * inverse))
        codes[g, first:first + len(x)] = np.clip(np.rint(x * inverse), -127, 127)
        scales[g] = s


def verify(x, tokens, cu, u, parents=None, q=None, temperature=None):
    """accepted, path, next tokens, one request and token at a time; x, q: fp64 arrays."""
    N, V = x.shape
    accepted, path, following = [], [-1] * N, []

    def dist(row, T):
        r = x[row]
        if np.isnan(r).any() or r.max() == np.inf or r.max() == -np.inf:
            return None
        if not T > 0:
            p = np.zeros(V)
            p[int(np.argmax(r))] = 1.0
            return p
        e = np.exp((r - r.max()) / T)
        return e / e.sum()

    for b in range(len(cu) - 1):
        t0, n = cu[b], cu[b + 1] - cu[b]
        if n <= 0:
            accepted.append(0), following.append(-1)
            continue
        T = 1.0 if temperature is None else float(temperature[b])
        last, kept = 0, [0]
        while True:
            p = dist(t0 + last, T)
            left, found = p, None
            if p is None:
                break
            most = n if parents is None else min(n, 64)
            for i in range(last + 1, most):
                up = i - 1 if parents is None else int(parents[t0 + i])
                if up != last:
                    continue
                t = int(tokens[t0 + i])
                if not 0 <= t < V:
                    if q is not None:
                        left = np.maximum(p - q[t0 + i], 0)
                    continue
                if q is not None:
                    if u[t0 + i] * q[t0 + i][t] < p[t]:
                        found = i
                    else:
                        left = np.maximum(p - q[t0 + i], 0)
                elif u[t0 + i] * (1 - (p.sum() - left.sum())) < left[t]:
                    found = i
                else:
                    left = left.copy()
                    left[t] = 0.0
                if found is not None:
                    break
            if found is None:
                break
            last = found
            kept.append(found)
        accepted.append(len(kept))
        for d, i in enumerate(kept):
            path[t0 + d] = i
        if p is None:
            following.append(-1)
            continue
        if not left.sum() > 0:
            left = p
        c = np.cumsum(left)
        following.append(int(np.argmax(c > u[t0] * c[-1])))
    return accepted, path, following
