"""Sampled speculative decoding over a cache of 8 bits, with a sliding window.

The model of verify_step.py, its caches int8 codes with a scale for each 16 tokens and
head, generates for a batch of requests.  Each step a draft of the model itself (its
likeliest tokens after the last verified row, as children of the last token, and one more
behind the first of them) is run as a tree; verify_draft accepts a branch and draws the next token,
keep_accepted moves the branch behind the context:

    plan_step, fused_qkv, qk_norm_rope, tree_attention, .., matmul_transB      the drafted trees
    verify_draft, keep_accepted                                              what stays

    python examples/sample_drafts.py

checks that with one token a step and temperature 0 the same tokens come out, as far as 8-bit
rounding leaves the likeliest token what it is.
"""
from __future__ import annotations

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import verify_step as V  # noqa: E402
from forge_amd import ops, step  # noqa: E402

WINDOW, SINKS = 96, 4


class Model(V.Model):
    """verify_step's model over caches of 8 bits and with a window."""

    def __init__(self, seed: int = 0, blocks: int = 64):
        super().__init__(seed, blocks)
        for w in self.layers:
            w["cache"] = step.paged_cache(blocks, V.BLOCK, V.KV_HEADS, V.HEAD_DIM, torch.int8)

    def forward(self, tokens, plan, block_table, lengths):
        def rms(x):
            return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)

        x = self.embedding[tokens.long()]
        for w in self.layers:
            k, v = w["cache"]
            qkv = ops.fused_qkv(rms(x), w["q"], w["k"], w["v"])
            q = step.qk_norm_rope(qkv, plan.positions, plan.slots, self.table, k, v,
                                  q_weight=self.norm, k_weight=self.norm)
            a = step.tree_attention(q, k, v, block_table, lengths, plan.cu, plan.masks, window=WINDOW, sinks=SINKS)
            x = x + ops.matmul_transB(a.flatten(1), w["o"])
            x = ops.ffn_down_residual(ops.ffn_up_fused(rms(x), w["gate"], w["up"]), w["down"], x)
        return ops.matmul_transB(rms(x), self.head)


class Requests(V.Requests):
    """Requests that keep some of a step's tokens: blocks behind what they keep are free again."""

    def keep(self, plan, new):
        self.lengths = self.lengths + new
        held = torch.arange(self.table.shape[1], device="cuda")[None] < ((self.lengths + V.BLOCK - 1) // V.BLOCK)[:, None]
        free = torch.ones(64, dtype=torch.bool, device="cuda")
        free[self.table[held].long()] = False
        self.free = free.nonzero()[:, 0].int()


def generate(prompts, steps, width, temperature, seed=0):
    """Tokens of each request after so many steps of drafts with `width` children of the last token."""
    dev = "cuda"
    model, B = Model(), len(prompts)
    g = torch.Generator(device=dev).manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    batch = Requests(B, columns=16)
    temps = torch.full((B,), float(temperature), device=dev)
    new = ints([len(p) for p in prompts])
    plan, logits = batch.run(model, ints(sum(prompts, [])), new)
    batch.keep(plan, new)
    ends = plan.cu[1:].long() - 1  # the prompts' last tokens: their rows alone, one token a request
    rows = logits[ends].contiguous()
    done = step.verify_draft(rows, torch.zeros(B, dtype=torch.int32, device=dev), ints(list(range(B + 1))),
                             torch.rand(B, generator=g, device=dev), temperature=temps)
    out = [[t] for t in done.next_tokens.tolist()]
    last, guess = done.next_tokens, rows
    for _ in range(steps):
        # the draft: the last token, the likeliest ones after the last known row, one behind the first
        likely = guess.topk(max(width, 1), -1).indices.int()
        tree, parents = [last[:, None]], [-1]
        if width:
            tree += [likely, likely[:, :1]]
            parents += [0] * width + [1]
        tokens = torch.cat(tree, 1)
        n = tokens.shape[1]
        plan, logits = batch.run(model, tokens.reshape(-1).contiguous(), ints([n] * B), parents=ints(parents * B))
        done = step.verify_draft(logits, tokens.reshape(-1).contiguous(), plan.cu, torch.rand(B * n, generator=g, device=dev),
                                 parents=ints(parents * B), temperature=temps)
        for w in model.layers:
            step.keep_accepted(*w["cache"], batch.table, batch.lengths, plan.cu, done.path, done.accepted)
        batch.keep(plan, done.accepted)
        path, accepted = done.path.view(B, n), done.accepted.tolist()
        for b in range(B):
            out[b] += [int(tokens[b, i]) for i in path[b, 1:accepted[b]].tolist()] + [int(done.next_tokens[b])]
        at = path.gather(1, done.accepted.long()[:, None] - 1)[:, 0].long()
        guess = logits.view(B, n, -1)[torch.arange(B, device=dev), at]
        last = done.next_tokens
    return out


def main() -> None:
    prompts = [[5, 17, 900, 3, 42], [7] * 150]
    drafted = generate(prompts, 12, 6, 1.0)
    print("tokens of 12 sampled steps:", [len(t) for t in drafted], "over caches of 8 bits")
    a, b = generate(prompts, 12, 6, 0.0), generate(prompts, 12, 0, 0.0)
    same = [next((i for i, (s, t) in enumerate(zip(x, y)) if s != t), min(len(x), len(y))) for x, y in zip(a, b)]
    print("first tokens at temperature 0 that are alike with drafts and without:", same)


if __name__ == "__main__":
    main()
