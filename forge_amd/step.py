"""Operators of one decoding or verifying step around the quantized matmuls.

A serving step over a paged key/value cache runs, with ``forge_amd.ops`` for
the projections::

    plan = plan_step(lengths, new_tokens, block_table, free_blocks, block_size, N, parents)
    for each layer:
        qkv = ops.fused_qkv(x, wq, wk, wv)
        q = qk_norm_rope(qkv, plan.positions, plan.slots, table, k_cache, v_cache)
        o = tree_attention(q, k_cache, v_cache, block_table, lengths, plan.cu, plan.masks)
        y = ops.matmul_transB(o.view(N, -1), wo)
        ...
    scores = token_logprobs(logits, targets, top=5)

They stand where the reference verifies drafted tokens
(src/inference/speculative.cpp:64) over its paged cache, with activations in
fp32 as everywhere here and caches in fp16 or bf16.  All arithmetic runs in
libforge_q.so (include/forge_step.h, which states the operators in full);
nothing waits for the GPU, and no length is needed on the host but the sum of
the new tokens.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _stream_ptr

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 100}


class StepPlan(NamedTuple):
    """What plan_step makes of a step (N tokens of B requests)."""
    cu: torch.Tensor         # int32 [B + 1]: request b's tokens are cu[b] .. cu[b + 1] - 1
    slots: torch.Tensor      # int32 [N]: each token's slot in the cache, -1: none
    positions: torch.Tensor  # int32 [N]: each token's position, its length + its depth
    masks: Optional[torch.Tensor]  # int64 [N]: the new tokens that a token sees, as bits (trees)
    info: torch.Tensor       # int32 [2]: blocks taken from the free ones, blocks that were missing


class TokenLogprobs(NamedTuple):
    """token_logprobs' results for M rows."""
    logprobs: Optional[torch.Tensor]      # fp32, targets' shape
    entropy: torch.Tensor                 # fp32 [M]
    top_logprobs: Optional[torch.Tensor]  # fp32 [M, top]
    top_tokens: Optional[torch.Tensor]    # int32 [M, top]


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise RuntimeError(what)


def _ints(name: str, t: torch.Tensor, shape, like: torch.Tensor, dtype=torch.int32):
    _need(t.dtype == dtype and t.is_contiguous() and t.device == like.device
          and tuple(t.shape) == tuple(shape),
          f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on {like.device}")
    return t.data_ptr()


def _table(name: str, t: torch.Tensor, rows: int, like: torch.Tensor) -> None:
    _need(t.dim() == 2 and t.shape[0] == rows and t.shape[1] >= 1 and t.dtype == torch.int32
          and t.device == like.device and t.stride(1) == 1 and t.stride(0) >= t.shape[1],
          f"{name} must be an int32 block table of {rows} rows on {like.device}")


def paged_cache(num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int,
                dtype: torch.dtype = torch.float16, device="cuda"):
    """Zeroed key and value caches [num_blocks, block_size, n_kv_heads, head_dim].
    A block's rows lie head by head in memory, so that a head's keys are read in
    long runs; any other order of the first three axes is accepted as well."""
    return tuple(torch.zeros((num_blocks, n_kv_heads, block_size, head_dim), dtype=dtype,
                             device=device).transpose(1, 2) for _ in range(2))


def _cache(name: str, k: torch.Tensor, v: torch.Tensor, like: torch.Tensor):
    _need(k.dim() == 4 and k.shape == v.shape and k.stride() == v.stride() and k.dtype == v.dtype
          and k.device == like.device and v.device == like.device,
          f"{name}: caches must be 4D [blocks, block size, kv heads, D], alike, on {like.device}")
    _need(k.dtype in (torch.float16, torch.bfloat16), f"{name}: caches must be fp16 or bf16")
    _need(k.stride(3) == 1, f"{name}: a cached head must be contiguous")
    return _TYPES[k.dtype], k.data_ptr(), v.data_ptr(), k.shape[0], k.shape[1], *k.stride()[:3]


def plan_step(lengths: torch.Tensor, new_tokens: torch.Tensor, block_table: torch.Tensor,
              free_blocks: torch.Tensor, block_size: int, n_tokens: int,
              parents: Optional[torch.Tensor] = None) -> StepPlan:
    """Slots, positions and masks of a step's n_tokens new tokens.

    lengths, new_tokens: int32 [B], each request's cached and new tokens; block_table:
    int32 [B, max blocks], into which the blocks that the new tokens need are
    entered, taken from free_blocks (int32 [F]) front to back; parents: int32
    [n_tokens], each drafted token's parent by its number within the request
    (-1: the context), at most 64 tokens a request; None: chains.  Rows past the
    last request's are padding (slot -1).  The call repeats itself: given the
    same lengths and free blocks it enters the same blocks."""
    _need(lengths.is_cuda and lengths.dim() == 1, "plan_step: lengths must be a 1D device tensor")
    B = lengths.shape[0]
    n = _ints("plan_step: lengths", lengths, (B,), lengths)
    t = _ints("plan_step: new_tokens", new_tokens, (B,), lengths)
    _table("plan_step: block_table", block_table, B, lengths)
    f = _ints("plan_step: free_blocks", free_blocks, (free_blocks.numel(),), lengths)
    p = None if parents is None else _ints("plan_step: parents", parents, (n_tokens,), lengths)
    # one allocation: cu, info, slots, positions
    out = lengths.new_empty((B + 3 + 2 * n_tokens,))
    cu, info, slots, positions = out.split((B + 1, 2, n_tokens, n_tokens))
    masks = None if parents is None else lengths.new_empty((n_tokens,), dtype=torch.int64)
    at = out.data_ptr()
    _lib.check(_lib.lib().fq_plan_step(
        n, t, p, B, n_tokens, block_size, block_table.data_ptr(), block_table.shape[1],
        block_table.stride(0), f, free_blocks.numel(), at, at + 4 * (B + 3),
        at + 4 * (B + 3 + n_tokens), None if masks is None else masks.data_ptr(), at + 4 * (B + 1),
        _stream_ptr(lengths)), "plan_step")
    return StepPlan(cu, slots, positions, masks, info)


def rope_table(positions: int, rot: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos and sin [positions, rot] (cos in the first half of a row) of the angles
    position * base^(-2i / rot), computed in 64 bits."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _vector(name: str, t: Optional[torch.Tensor], n: int, like: torch.Tensor):
    if t is None:
        return None
    _need(t.dtype == torch.float32 and t.is_contiguous() and t.numel() == n
          and t.device == like.device, f"{name} must be {n} contiguous fp32 values on {like.device}")
    return t.data_ptr()


def qk_norm_rope(qkv: torch.Tensor, positions: torch.Tensor, slots: torch.Tensor,
                 table: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, *,
                 bias: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                 k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> torch.Tensor:
    """Queries [N, hq, D] of fused_qkv's rows; keys and values go to the caches.

    qkv: fp32 [N, (hq + 2 hkv) D], rows any distance apart; table: rope_table's cos
    and sin, whose width is the number of rotated elements of a head; bias: fp32,
    added to each row first; q_weight, k_weight: fp32 [D], the heads' RMS norms
    (none: not normalized); interleaved: pairs (2i, 2i + 1) instead of (i, i + rot / 2).
    Tokens whose slot is -1 leave the caches as they are."""
    _need(qkv.dim() == 2 and qkv.is_cuda and qkv.dtype == torch.float32
          and (qkv.stride(1) == 1 or qkv.shape[1] == 1),
          "qk_norm_rope: qkv must be a 2D fp32 device tensor of contiguous rows")
    type_, k, v, nb, bs, sb, st, sh = _cache("qk_norm_rope", k_cache, v_cache, qkv)
    N, width = qkv.shape
    hkv, D = k_cache.shape[2:]
    hq = width // D - 2 * hkv
    _need(width % D == 0 and hq >= 1 and hq % hkv == 0,
          f"qk_norm_rope: rows of {width} do not hold heads of {D} for {hkv} kv heads")
    _need(table.dim() == 2 and table.dtype == torch.float32 and table.is_contiguous()
          and table.device == qkv.device, "qk_norm_rope: table must be a contiguous fp32 [positions, rot]")
    q = qkv.new_empty((N, hq, D))
    _lib.check(_lib.lib().fq_qk_norm_rope(
        qkv.data_ptr(), qkv.stride(0) if N > 1 else width, N, hq, hkv, D, table.shape[1],
        1 if interleaved else 0, _vector("qk_norm_rope: bias", bias, width, qkv),
        _vector("qk_norm_rope: q_weight", q_weight, D, qkv),
        _vector("qk_norm_rope: k_weight", k_weight, D, qkv), eps,
        _ints("qk_norm_rope: positions", positions, (N,), qkv),
        _ints("qk_norm_rope: slots", slots, (N,), qkv), table.data_ptr(), table.shape[0],
        q.data_ptr(), type_, k, v, nb, bs, sb, st, sh, _stream_ptr(qkv)), "qk_norm_rope")
    return q


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor,
                   masks: Optional[torch.Tensor] = None, *, max_new: Optional[int] = None,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the step's tokens, fp32 [N, hq, D].

    q: fp32 [N, hq, D], tokens any distance apart; lengths: int32 [B], the cached tokens
    before this step; cu, masks: plan_step's (masks None: chains, a token sees
    the ones before it and itself); the new tokens' keys and values are in the
    caches already.  A token sees all of its request's cached tokens.  max_new:
    the most new tokens of one request where the caller knows it (speed only);
    scale: D^-0.5 unless given."""
    _need(q.dim() == 3 and q.is_cuda and q.dtype == torch.float32,
          "tree_attention: q must be a 3D fp32 device tensor")
    N, hq, D = q.shape
    _need(q.stride(2) == 1 and (hq == 1 or q.stride(1) == D),
          "tree_attention: a token's queries must be contiguous")
    type_, k, v, nb, bs, sb, st, sh = _cache("tree_attention", k_cache, v_cache, q)
    hkv = k_cache.shape[2]
    _need(k_cache.shape[3] == D and hkv >= 1 and hq % hkv == 0,
          f"tree_attention: {hq} heads of {D} do not share {hkv} kv heads of {k_cache.shape[3]}")
    B = lengths.shape[0] if lengths.dim() == 1 else -1
    n = _ints("tree_attention: lengths", lengths, (B,), q)
    c = _ints("tree_attention: cu", cu, (B + 1,), q)
    m = None if masks is None else _ints("tree_attention: masks", masks, (N,), q, torch.int64)
    _table("tree_attention: block_table", block_table, B, q)
    out = q.new_empty((N, hq, D))
    _lib.check(_lib.lib().fq_tree_attention(
        q.data_ptr(), q.stride(0) if N > 1 else hq * D, n, c, m, B, N,
        N if max_new is None else max_new, hq, hkv, D, D ** -0.5 if scale is None else scale,
        type_, k, v, nb, bs, sb, st, sh, block_table.data_ptr(), block_table.shape[1],
        block_table.stride(0), out.data_ptr(), _stream_ptr(q)), "tree_attention")
    return out


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None,
                   top: int = 0) -> TokenLogprobs:
    """Log probabilities of targets (int32 [M] or [M, J]) under softmax(logits) (fp32,
    fp16 or bf16 [M, V], rows any distance apart), each row's entropy, and its top
    largest logits (at most 64; ties: the lowest token) with their log probabilities."""
    _need(logits.dim() == 2 and logits.is_cuda and logits.dtype in _TYPES
          and (logits.stride(1) == 1 or logits.shape[1] == 1),
          "token_logprobs: logits must be a 2D fp32, fp16 or bf16 device tensor of contiguous rows")
    M, V = logits.shape
    t, J, lp, tl, tt = None, 0, None, None, None
    if targets is not None:
        _need(targets.dim() in (1, 2), "token_logprobs: targets must be [M] or [M, J]")
        J = 1 if targets.dim() == 1 else targets.shape[1]
        t = _ints("token_logprobs: targets", targets, (M,) if targets.dim() == 1 else (M, J), logits)
        lp = logits.new_empty(targets.shape, dtype=torch.float32)
    entropy = logits.new_empty((M,), dtype=torch.float32)
    if top:
        _need(0 < top <= min(64, V), f"token_logprobs: top must be at most {min(64, V)}")
        tl = logits.new_empty((M, top), dtype=torch.float32)
        tt = logits.new_empty((M, top), dtype=torch.int32)
    _lib.check(_lib.lib().fq_token_logprobs(
        logits.data_ptr(), _TYPES[logits.dtype], logits.stride(0) if M > 1 else V, M, V, t, J, top,
        None if lp is None else lp.data_ptr(), entropy.data_ptr(),
        None if tl is None else tl.data_ptr(), None if tt is None else tt.data_ptr(),
        _stream_ptr(logits)), "token_logprobs")
    return TokenLogprobs(lp, entropy, tl, tt)


def reserve(device="cuda") -> None:
    """Sizes the current stream's workspace for every call here, before a capture
    into a HIP graph (the first call on a stream does it as well)."""
    st = torch.cuda.current_stream(torch.device(device)).cuda_stream
    with torch.cuda.device(torch.device(device)):
        _lib.check(_lib.lib().fq_reserve_step(st), "reserve")
