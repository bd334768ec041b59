"""Sampled speculative decoding over a cache of 8 bits, with a sliding window.

The model of verify_step.py, its caches int8 codes with a scale for each 16 tokens and
head, generates for a batch of requests.  Each step a draft of the model itself (its
likeliest tokens after the last verified row, as children of the last token, and one more
behind the first of them) is run as a tree; verify_draft accepts a branch and draws the next token,
keep_accepted moves the branch behind the context:

    plan_step, fused_qkv, qk_norm_rope, tree_attention, .., matmul_transB      the drafted trees
    verify_draft, keep_accepted                                              what stays

    python examples/sample_drafts.py

samples, then checks at temperature 0, over caches of 16 and of 8 bits, that drafted steps say of each
token what steps of one token say: drafts in which the tokens that are taken stand behind others, so that
each step moves a branch.
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
    """verify_step's model over caches of that type and with a window."""

    def __init__(self, seed: int = 0, blocks: int = 64, cache: torch.dtype = torch.int8):
        super().__init__(seed, blocks)
        for w in self.layers:
            w["cache"] = step.paged_cache(blocks, V.BLOCK, V.KV_HEADS, V.HEAD_DIM, cache)

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


def generate(prompts, steps, width, temperature, seed=0, cache=torch.int8, known=None):
    """Tokens of each request after so many steps of drafts with `width` children of the last token, and
    the logits that each was drawn from.  known: tokens of each request to be drafted as well, behind those."""
    dev = "cuda"
    model, B = Model(cache=cache), len(prompts)
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
    out, drawn = [[t] for t in done.next_tokens.tolist()], [[r] for r in rows]
    last, guess = done.next_tokens, rows
    for _ in range(steps):
        # the draft: the last token, the likeliest ones after the last known row, one behind the first
        likely = guess.topk(max(width, 1), -1).indices.int()
        tree, parents = [last[:, None]], [-1]
        if width:
            tree += [likely, likely[:, :1]]
            parents += [0] * width + [1]
        if known:
            after = [(t + [0, 0])[len(o):len(o) + 2] if len(o) < len(t) else [0, 0] for t, o in zip(known, out)]
            tree.append(ints(after))
            parents += [0, len(parents)]
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
            kept = path[b, :accepted[b]].tolist()
            out[b] += [int(tokens[b, i]) for i in kept[1:]] + [int(done.next_tokens[b])]
            drawn[b] += [logits.view(B, n, -1)[b, i] for i in kept]
        at = path.gather(1, done.accepted.long()[:, None] - 1)[:, 0].long()
        guess = logits.view(B, n, -1)[torch.arange(B, device=dev), at]
        last = done.next_tokens
    return out, drawn


def compare(prompts, steps, cache):
    """Steps of one token, then drafted ones that hold what those said, at temperature 0: how many first tokens
    are alike, of how many, and how far the logits of those (and of the first that is not) are apart."""
    alone, say = generate(prompts, 2 * steps, 0, 0.0, cache=cache)
    drafted, also = generate(prompts, steps, 3, 0.0, cache=cache, known=alone)
    alike, most, worst = [], [], 0.0
    for x, y, r, s in zip(alone, drafted, say, also):
        most.append(min(len(x), len(y)))
        alike.append(next((i for i, (t, u) in enumerate(zip(x, y)) if t != u), most[-1]))
        for a, b in list(zip(r, s))[:alike[-1] + 1]:
            worst = max(worst, float((a - b).norm() / a.norm()))
    return alike, most, worst


def main():
    prompts = [[5, 17, 900, 3, 42], [7] * 150]
    drafted, _ = generate(prompts, 12, 6, 1.0)
    print("tokens of 12 sampled steps:", [len(t) for t in drafted], "over caches of 8 bits")
    results = {}
    # In 16 bits only the steps' sizes round differently.  In 8 bits the two runs' groups have scales of their own: an
    # element is off by half a 127th of its group's largest (four times its root mean square or so) in each
    # run, 1 % of that root mean square, a key's score and a value by as much, and these add up.
    for cache, bound in ((torch.float16, 5e-3), (torch.int8, 5e-2)):
        alike, most, worst = results[cache] = compare(prompts, 12, cache)
        print(f"{cache}: {alike} of {most} tokens alike with drafts and without, logits {worst:.1e} apart")
        assert worst < bound and min(most) > 13, "drafted steps say something else"
    return results


if __name__ == "__main__":
    main()
