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

or, where drafted tokens are sampled::

    done = verify_draft(logits, tokens, plan.cu, uniforms, parents=parents)
    for each layer:
        keep_accepted(k_cache, v_cache, block_table, lengths, plan.cu, done.path, done.accepted)
    lengths += done.accepted

They stand where the reference verifies drafted tokens
(src/inference/speculative.cpp:64) over its paged cache, with activations in
fp32 as everywhere here and caches in fp16 or bf16, or in 8 bits (Cache8).  All arithmetic runs in
libforge_q.so (include/forge_step.h, which states the operators in full);
nothing waits for the GPU, and no length is needed on the host but the sum of
the new tokens.  examples/verify_step.py runs a small model through them, examples/sample_drafts.py the
sampling of drafted trees over a cache of 8 bits.
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


class Cache8(NamedTuple):
    """Keys or values in 8 bits: codes times the scale of their 16 tokens and kv head.
    What takes k_cache and v_cache takes a pair of these in their place."""
    codes: torch.Tensor   # int8 [num_blocks, block_size, n_kv_heads, head_dim]
    scales: torch.Tensor  # fp32 [num_blocks, n_kv_heads, block_size / 16]


class Verified(NamedTuple):
    """verify_draft's results for B requests of N tokens."""
    accepted: torch.Tensor     # int32 [B]: accepted tokens, the known one included
    path: torch.Tensor         # int32 [N]: path[cu[b] + d] is the number of the d-th accepted one, -1 behind
    next_tokens: torch.Tensor  # int32 [B]: the token after the last accepted one; -1: none


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
    long runs; any other order of the first three axes is accepted as well.  dtype int8: a
    pair of Cache8, half the bytes; a head's tokens 16 n .. 16 n + 15 share a scale."""
    def cache():
        data = torch.zeros((num_blocks, n_kv_heads, block_size, head_dim), dtype=dtype,
                           device=device).transpose(1, 2)
        if dtype != torch.int8:
            return data
        return Cache8(data, torch.zeros((num_blocks, n_kv_heads, block_size // 16), device=device))

    return cache(), cache()


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
    Tokens whose slot is -1 leave the caches as they are.

    Into a Cache8 the tokens of a request go as plan_step's slots have them, next to each other.  16
    tokens and a kv head share a scale, the largest magnitude over 127; a token that
    needs a larger one than its group has gives the group that, and the codes held are
    rounded again.  (A drafted token that is refused later has its part in that scale, until the
    group's first slot is written again.)  Infinite elements are held to the largest finite one of the group, NaN is 0."""
    return _native().rope(qkv, positions, slots, table, k_cache, v_cache, bias, q_weight, k_weight, eps,
                          interleaved, _stream(qkv))


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                   block_table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor,
                   masks: Optional[torch.Tensor] = None, *, max_new: Optional[int] = None,
                   scale: Optional[float] = None, window: Optional[int] = None, sinks: int = 0) -> torch.Tensor:
    """Attention of the step's tokens, fp32 [N, hq, D].

    q: fp32 [N, hq, D], tokens any distance apart; lengths: int32 [B], the cached tokens
    before this step; cu, masks: plan_step's (masks None: chains, a token sees
    the ones before it and itself); the new tokens' keys and values are in the
    caches already.  A token sees all of its request's cached tokens; what a table entry
    that is no block of the caches (-1: plan_step had none left) would hold is not
    there, so that info[1] of the plan, where it is not 0, says that answers lack it.  max_new:
    the most new tokens of one request where the caller knows it (it chooses how many
    rows a tile has; without it their average is taken); scale: D^-0.5 unless given.

    window: of the keys above, a token sees those of the window positions up to its own and
    those of the request's first sinks positions (a drafted token's position is that of plan_step);
    what no token of the call sees is not read.

    Over a Cache8 a query's elements count to 24 bits of the largest of its head's."""
    return _native().attention(q, k_cache, v_cache, block_table, lengths, cu, masks, max_new, scale,
                               window, sinks, _stream(q))


_READ = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 100}


def read_cache(k_cache: Cache8, v_cache: Cache8, block_table: torch.Tensor, starts: torch.Tensor,
               n_tokens: int, *, first: Optional[torch.Tensor] = None,
               dtype: torch.dtype = torch.float16):
    """Keys and values [n_tokens, kv heads, D] of caches of 8 bits in fp16, bf16 or fp32.

    Rows starts[b] .. starts[b + 1] - 1 (int32 [B + 1], prefix sums) are the tokens of request
    b from its number first[b] (int32 [B]; none: its first) on.  Tokens whose block the
    table does not have, and rows past the last request's, are zeros."""
    if dtype not in _READ:
        raise RuntimeError("read_cache: dtype must be fp16, bf16 or fp32")
    return _native().read(k_cache, v_cache, block_table, starts, n_tokens, _READ[dtype], first, _stream(starts))


def verify_draft(logits: torch.Tensor, tokens: torch.Tensor, cu: torch.Tensor, uniforms: torch.Tensor, *,
                 parents: Optional[torch.Tensor] = None, draft_probs: Optional[torch.Tensor] = None,
                 temperature: Optional[torch.Tensor] = None) -> Verified:
    """Which drafted tokens a step's logits accept, and each request's next token.

    The step's tokens (int32 [N], plan_step's cu) are each request's last sampled token, which
    is accepted, and drafted ones behind it; logits (fp32, fp16 or bf16 [N, V], rows any
    distance apart) are what the model says after each; uniforms: fp32 [N] in [0, 1).
    parents: as plan_step's (None: chains).  The accepted tokens and the next one
    are distributed as tokens sampled one by one from softmax(logits / temperature), whatever was
    drafted: token i is tried with uniforms[i] against what its refused siblings left, the next token
    is drawn with the request's first one.  draft_probs: fp32 [N, V], row i the distribution that token i of a
    chain was drawn from; without it drafted tokens are taken as given.  temperature: fp32 [B],
    finite (None: 1; 0: the largest logit, of equal ones the lowest token).  With one
    token a request this samples the next one.

    A row with a NaN or +inf logit or nothing but -inf ends its request with next token -1."""
    return Verified(*_native().verify(logits, tokens, cu, uniforms, parents, draft_probs, temperature,
                                      _stream(logits)))


def keep_accepted(k_cache, v_cache, block_table: torch.Tensor, lengths: torch.Tensor, cu: torch.Tensor,
                  path: torch.Tensor, accepted: torch.Tensor) -> None:
    """Moves verify_draft's accepted tokens behind the context: their keys and values, in caches of
    any type, go to the slots of numbers lengths[b], lengths[b] + 1, .., after which
    lengths + accepted are the requests' lengths.  lengths: those before the step.  Chains stay where they are.
    In a Cache8 a moved token's codes are rounded again where its new group has another scale."""
    _native().keep(k_cache, v_cache, block_table, lengths, cu, path, accepted, _stream(lengths))


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
