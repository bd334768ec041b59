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


def _refuse(what: str):
    raise RuntimeError(what)


# The checks below format a message only where they refuse: they are most of what a
# call costs the host (17 -> 9 us a call with the messages made in advance).
def _ints(name: str, t: torch.Tensor, shape, dev: int, dtype=torch.int32) -> int:
    """t's address, if it is a contiguous tensor of that type and shape on GPU dev."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on cuda:{dev}")
    return t.data_ptr()


def _table(name: str, t: torch.Tensor, rows: int, dev: int):
    """A block table's address, columns and distance of rows."""
    if t.dim() == 2 and t.dtype is torch.int32 and t.get_device() == dev:
        n, cols = t.shape
        stride, one = t.stride()
        if n == rows and cols >= 1 and (one == 1 or cols == 1) and (stride >= cols or n == 1):
            return t.data_ptr(), cols, max(stride, cols)
    _refuse(f"{name} must be an int32 block table of {rows} rows on cuda:{dev}")


def paged_cache(num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int,
                dtype: torch.dtype = torch.float16, device="cuda"):
    """Zeroed key and value caches [num_blocks, block_size, n_kv_heads, head_dim].
    A block's rows lie head by head in memory, so that a head's keys are read in
    long runs; any other order of the first three axes is accepted as well."""
    return tuple(torch.zeros((num_blocks, n_kv_heads, block_size, head_dim), dtype=dtype,
                             device=device).transpose(1, 2) for _ in range(2))


def _cache(name: str, k: torch.Tensor, v: torch.Tensor, dev: int):
    if (k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype is not v.dtype
            or k.get_device() != dev or v.get_device() != dev):
        _refuse(f"{name}: caches must be 4D [blocks, block size, kv heads, D], alike, on cuda:{dev}")
    if k.dtype is not torch.float16 and k.dtype is not torch.bfloat16:
        _refuse(f"{name}: caches must be fp16 or bf16")
    nb, bs, hkv, D = k.shape
    sb, st, sh, one = k.stride()
    if one != 1 and D != 1:
        _refuse(f"{name}: a cached head must be contiguous")
    return _TYPES[k.dtype], k.data_ptr(), v.data_ptr(), nb, bs, sb, st, sh, hkv, D


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
    if not lengths.is_cuda or lengths.dim() != 1:
        _refuse("plan_step: lengths must be a 1D device tensor")
    B, dev, N = lengths.shape[0], lengths.get_device(), n_tokens
    n = _ints("plan_step: lengths", lengths, (B,), dev)
    t = _ints("plan_step: new_tokens", new_tokens, (B,), dev)
    table, cols, stride = _table("plan_step: block_table", block_table, B, dev)
    n_free = free_blocks.numel()
    f = _ints("plan_step: free_blocks", free_blocks, (n_free,), dev)
    p = masks = m = None
    if parents is not None:
        p = _ints("plan_step: parents", parents, (N,), dev)
        masks = torch.empty_like(parents, dtype=torch.int64)
        m = masks.data_ptr()
    out = lengths.new_empty((B + 3 + 2 * N,))  # one allocation
    at = out.data_ptr()
    _lib.check(_lib.lib().fq_plan_step(
        n, t, p, B, N, block_size, table, cols, stride, f, n_free, at, at + 4 * (B + 3),
        at + 4 * (B + 3 + N), m, at + 4 * (B + 1), _stream_ptr(lengths)), "plan_step")
    cu, info, slots, positions = out.split_with_sizes((B + 1, 2, N, N))
    return StepPlan(cu, slots, positions, masks, info)


def rope_table(positions: int, rot: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos and sin [positions, rot] (cos in the first half of a row) of the angles
    position * base^(-2i / rot), computed in 64 bits."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _vector(name: str, t: Optional[torch.Tensor], n: int, dev: int):
    if t is None:
        return None
    if t.dtype is not torch.float32 or t.numel() != n or t.get_device() != dev or not t.is_contiguous():
        _refuse(f"{name} must be {n} contiguous fp32 values on cuda:{dev}")
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
    if (qkv.dim() != 2 or not qkv.is_cuda or qkv.dtype is not torch.float32
            or (qkv.stride(1) != 1 and qkv.shape[1] != 1)):
        _refuse("qk_norm_rope: qkv must be a 2D fp32 device tensor of contiguous rows")
    dev = qkv.get_device()
    type_, k, v, nb, bs, sb, st, sh, hkv, D = _cache("qk_norm_rope", k_cache, v_cache, dev)
    N, width = qkv.shape
    hq = width // D - 2 * hkv if D else 0
    if hq < 1 or width % D or hkv < 1 or hq % hkv:
        _refuse(f"qk_norm_rope: rows of {width} do not hold heads of {D} for {hkv} kv heads")
    if (table.dim() != 2 or table.dtype is not torch.float32 or not table.is_contiguous()
            or table.get_device() != dev):
        _refuse(f"qk_norm_rope: table must be a contiguous fp32 [positions, rot] on cuda:{dev}")
    rows, rot = table.shape
    q = qkv.new_empty((N, hq, D))
    _lib.check(_lib.lib().fq_qk_norm_rope(
        qkv.data_ptr(), qkv.stride(0) if N > 1 else width, N, hq, hkv, D, rot,
        1 if interleaved else 0, _vector("qk_norm_rope: bias", bias, width, dev),
        _vector("qk_norm_rope: q_weight", q_weight, D, dev),
        _vector("qk_norm_rope: k_weight", k_weight, D, dev), eps,
        _ints("qk_norm_rope: positions", positions, (N,), dev),
        _ints("qk_norm_rope: slots", slots, (N,), dev), table.data_ptr(), rows,
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
    if q.dim() != 3 or not q.is_cuda or q.dtype is not torch.float32:
        _refuse("tree_attention: q must be a 3D fp32 device tensor")
    N, hq, D = q.shape
    ldq, sq, one = q.stride()
    if one != 1 or (hq != 1 and sq != D):
        _refuse("tree_attention: a token's queries must be contiguous")
    dev = q.get_device()
    type_, k, v, nb, bs, sb, st, sh, hkv, Dk = _cache("tree_attention", k_cache, v_cache, dev)
    if Dk != D or hkv < 1 or hq % hkv:
        _refuse(f"tree_attention: {hq} heads of {D} do not share {hkv} kv heads of {Dk}")
    B = lengths.numel()
    n = _ints("tree_attention: lengths", lengths, (B,), dev)
    c = _ints("tree_attention: cu", cu, (B + 1,), dev)
    m = None if masks is None else _ints("tree_attention: masks", masks, (N,), dev, torch.int64)
    table, cols, stride = _table("tree_attention: block_table", block_table, B, dev)
    out = q.new_empty((N, hq, D))
    _lib.check(_lib.lib().fq_tree_attention(
        q.data_ptr(), ldq if N > 1 else hq * D, n, c, m, B, N, N if max_new is None else max_new, hq,
        hkv, D, D ** -0.5 if scale is None else scale, type_, k, v, nb, bs, sb, st, sh, table, cols,
        stride, out.data_ptr(), _stream_ptr(q)), "tree_attention")
    return out


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None,
                   top: int = 0) -> TokenLogprobs:
    """Log probabilities of targets (int32 [M] or [M, J]) under softmax(logits) (fp32,
    fp16 or bf16 [M, V], rows any distance apart), each row's entropy, and its top
    largest logits (at most 64; ties: the lowest token) with their log probabilities."""
    if (logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _TYPES
            or (logits.stride(1) != 1 and logits.shape[1] != 1)):
        _refuse("token_logprobs: logits must be a 2D fp32, fp16 or bf16 device tensor of contiguous rows")
    M, V = logits.shape
    J, t, lp, l, tl, tt, a, b = 0, None, None, None, None, None, None, None
    if targets is not None:
        if targets.dim() not in (1, 2):
            _refuse("token_logprobs: targets must be [M] or [M, J]")
        J = 1 if targets.dim() == 1 else targets.shape[1]
        t = _ints("token_logprobs: targets", targets, (M, J)[:targets.dim()], logits.get_device())
        lp = torch.empty_like(targets, dtype=torch.float32)
        l = lp.data_ptr()
    entropy = logits.new_empty((M,), dtype=torch.float32)
    if top:
        if not 0 < top <= min(64, V):
            _refuse(f"token_logprobs: top must be at most {min(64, V)}")
        tl = logits.new_empty((M, top), dtype=torch.float32)
        tt = logits.new_empty((M, top), dtype=torch.int32)
        a, b = tl.data_ptr(), tt.data_ptr()
    _lib.check(_lib.lib().fq_token_logprobs(
        logits.data_ptr(), _TYPES[logits.dtype], logits.stride(0) if M > 1 else V, M, V, t, J, top, l,
        entropy.data_ptr(), a, b, _stream_ptr(logits)), "token_logprobs")
    return TokenLogprobs(lp, entropy, tl, tt)


def reserve(device="cuda") -> None:
    """Sizes the current stream's workspace for every call here, before a capture
    into a HIP graph (the first call on a stream does it as well)."""
    st = torch.cuda.current_stream(torch.device(device)).cuda_stream
    with torch.cuda.device(torch.device(device)):
        _lib.check(_lib.lib().fq_reserve_step(st), "reserve")
