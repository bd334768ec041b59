"""Plain 64-bit implementations of the step operators (include/forge_step.h),
written from their definitions, one request, head and row at a time."""
from __future__ import annotations

import numpy as np
import torch


def plan(lengths, new, parents, table, free, bs, N):
    """cu, slots, positions, masks, info and the table after the step, as lists / arrays."""
    B, cols = table.shape
    table = table.copy()
    cu, slots, positions, masks = [0], [-1] * N, [0] * N, [0] * N
    at = taken = missing = 0
    for b in range(B):
        ln, n = max(0, int(lengths[b])), max(0, int(new[b]))
        have, want = -(-ln // bs), -(-(ln + n) // bs)
        for c in range(have, want):
            if c < cols and at < len(free):
                table[b, c] = free[at]
                taken += 1
            else:
                missing += 1
                if c < cols:
                    table[b, c] = -1
            if c < cols:
                at += 1
        seen = {}
        for i in range(n):
            t = cu[-1] + i
            if t >= N:
                break
            m, depth = 1 << i, i
            if parents is not None:
                if i >= 64:
                    positions[t] = ln + 64
                    continue
                p = int(parents[t])
                p = p if 0 <= p < i else -1
                m |= seen.get(p, 0)
                depth = bin(m).count("1") - 1
            seen[i] = m
            masks[t] = m - (1 << 64) if m >> 63 and parents is not None else m
            positions[t] = ln + depth
            c = (ln + i) // bs
            if c < cols and table[b, c] >= 0:
                slots[t] = int(table[b, c]) * bs + (ln + i) % bs
        cu.append(cu[-1] + n)
    return cu, slots, positions, masks, [taken, missing], table


def norm_rope(x, hq, hkv, D, rot, interleaved, bias, qw, kw, eps, positions, table):
    """Heads [N, hq + 2 hkv, D] in fp64: normed and rotated queries and keys, values."""
    x = x.astype(np.float64)
    if bias is not None:
        x = x + bias.astype(np.float64)
    h = x.reshape(len(x), hq + 2 * hkv, D).copy()
    for w, lo, hi in ((qw, 0, hq), (kw, hq, hq + hkv)):
        if w is not None:
            part = h[:, lo:hi]
            h[:, lo:hi] = part / np.sqrt((part ** 2).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    for n, p in enumerate(positions):
        if not 0 <= p < len(table):
            h[n, :hq + hkv] = np.nan
            continue
        cos, sin = (table[p].astype(np.float64)[i * (rot // 2):(i + 1) * (rot // 2)] for i in (0, 1))
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        u, v = h[n, :hq + hkv, a].copy(), h[n, :hq + hkv, b].copy()
        h[n, :hq + hkv, a] = u * cos - v * sin
        h[n, :hq + hkv, b] = v * cos + u * sin
    return h


def attention(q, k_cache, v_cache, table, lengths, cu, masks, scale):
    """fp64 [N, hq, D] of the caches' values as they are; masked keys take no part."""
    N, hq, D = q.shape
    bs, hkv = k_cache.shape[1:3]
    out = torch.zeros((N, hq, D), dtype=torch.float64)
    for b in range(len(lengths)):
        ln, t0, n = int(lengths[b]), int(cu[b]), int(cu[b + 1]) - int(cu[b])
        if n == 0:
            continue
        keys = ln + n
        pages = table[b, :-(-keys // bs)].long()
        k = k_cache[pages].flatten(0, 1)[:keys].cpu().double()
        v = v_cache[pages].flatten(0, 1)[:keys].cpu().double()
        j = torch.arange(n)
        for i in range(n):
            if masks is None:
                see = j <= i
            else:
                m = int(masks[t0 + i])
                see = torch.tensor([c < 64 and (m >> c) & 1 == 1 for c in range(n)])
            idx = torch.cat([torch.arange(ln), ln + j[see]])
            if len(idx) == 0:
                continue
            kk = k[idx].repeat_interleave(hq // hkv, 1)  # [keys, hq, D]
            vv = v[idx].repeat_interleave(hq // hkv, 1)
            s = (q[t0 + i].cpu().double()[None] * kk).sum(-1) * scale
            out[t0 + i] = (torch.softmax(s, 0)[..., None] * vv).sum(0)
    return out


def logprobs(x, targets, top):
    """log p of targets, entropy, top tokens and their log p, in fp64."""
    x = x.double().cpu().numpy()
    M, V = x.shape
    lp = np.full((M, V), np.nan)
    H = np.full(M, np.nan)
    tokens = np.zeros((M, top), dtype=np.int64)
    for m in range(M):
        r = x[m]
        if not np.isnan(r).any() and r.max() != np.inf and r.max() != -np.inf:
            e = np.exp(r - r.max())
            lp[m] = r - r.max() - np.log(e.sum())
            p = e / e.sum()
            H[m] = -(p[p > 0] * np.log(p[p > 0])).sum()
        nan = np.isnan(r)
        order = np.lexsort((np.arange(V), -np.where(nan, 0.0, r), ~nan))
        tokens[m] = order[:top]
    t = targets.reshape(M, -1).astype(np.int64)
    tl = np.where((t >= 0) & (t < V), np.take_along_axis(lp, np.clip(t, 0, V - 1), 1), np.nan)
    return tl.reshape(targets.shape), H, tokens, np.take_along_axis(lp, tokens, 1)
