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
the new tokens.  examples/verify_step.py runs a small model through them.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib
from .ops import _stream_ptr


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


def _native():
    """The host side of these functions (csrc/fq_step_py.cpp); like the library it has no
    fallback."""
    global _n
    if _n is None:
        try:
            from . import _step
        except ImportError as e:
            raise ImportError("forge_amd/_step.so is missing or does not load: build it with "
                              f"`python -m forge_amd.build` ({e})") from e
        _n = _step
    return _n


_n = None


def _stream(t) -> int:
    return _stream_ptr(t) if isinstance(t, torch.Tensor) and t.is_cuda else 0


def paged_cache(num_blocks: int, block_size: int, n_kv_heads: int, head_dim: int,
                dtype: torch.dtype = torch.float16, device="cuda"):
    """Zeroed key and value caches [num_blocks, block_size, n_kv_heads, head_dim].
    A block's rows lie head by head in memory, so that a head's keys are read in
    long runs; any other order of the first three axes is accepted as well."""
    return tuple(torch.zeros((num_blocks, n_kv_heads, block_size, head_dim), dtype=dtype,
                             device=device).transpose(1, 2) for _ in range(2))


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
    return StepPlan(*_native().plan(lengths, new_tokens, block_table, free_blocks, block_size, n_tokens,
                                    parents, _stream(lengths)))


def rope_table(positions: int, rot: int, base: float = 10000.0, device="cuda") -> torch.Tensor:
    """cos and sin [positions, rot] (cos in the first half of a row) of the angles
    position * base^(-2i / rot), computed in 64 bits."""
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=device)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * base ** (-i / rot)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


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
    return _native().rope(qkv, positions, slots, table, k_cache, v_cache, bias, q_weight, k_weight, eps,
                          interleaved, _stream(qkv))


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor,
                   masks: Optional[torch.Tensor] = None, *, max_new: Optional[int] = None,
                   scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the step's tokens, fp32 [N, hq, D].

    q: fp32 [N, hq, D], tokens any distance apart; lengths: int32 [B], the cached tokens
    before this step; cu, masks: plan_step's (masks None: chains, a token sees
    the ones before it and itself); the new tokens' keys and values are in the
    caches already.  A token sees all of its request's cached tokens; what a table entry
    that is no block of the caches (-1: plan_step had none left) would hold is not
    there, so that info[1] of the plan, where it is not 0, says that answers lack it.  max_new:
    the most new tokens of one request where the caller knows it (it chooses how many
    rows a tile has; without it their average is taken); scale: D^-0.5 unless given."""
    return _native().attention(q, k_cache, v_cache, block_table, lengths, cu, masks, max_new, scale,
                               _stream(q))


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None,
                   top: int = 0) -> TokenLogprobs:
    """Log probabilities of targets (int32 [M] or [M, J]) under softmax(logits) (fp32,
    fp16 or bf16 [M, V], rows any distance apart), each row's entropy, and its top
    largest logits (at most 64; ties: the lowest token) with their log probabilities."""
    return TokenLogprobs(*_native().logprobs(logits, targets, top, _stream(logits)))


def reserve(device="cuda") -> None:
    """Sizes the current stream's workspace for every call here, before a capture
    into a HIP graph (the first call on a stream does it as well)."""
    st = torch.cuda.current_stream(torch.device(device)).cuda_stream
    with torch.cuda.device(torch.device(device)):
        _lib.check(_lib.lib().fq_reserve_step(st), "reserve")
