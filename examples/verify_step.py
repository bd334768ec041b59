"""Speculative decoding's verification, one step of a small quantized model.

Each request has a context in a paged cache and a tree of drafted tokens.  One
step runs all drafted tokens of all requests through the model at once and
accepts, from the root of each tree, the longest branch whose tokens the
model itself finds most likely:

    plan_step       blocks, slots, positions and masks of the drafted tokens
    fused_qkv, qk_norm_rope, tree_attention, matmul_transB, ffn_up_fused,
    ffn_down_residual                                        in every layer
    matmul_transB, token_logprobs                            over the vocabulary

    python examples/verify_step.py

runs it on random Q4_0 / Q8_0 weights and checks that a tree gives each token
what its own branch, decoded token by token, gives it.  It ends with what is
accepted: before the next step a program moves the accepted branch's keys and
values to the slots right behind the context (a branch that is not the draft's first
tokens lies apart in the cache), or runs its tokens once more as a chain.
"""
from __future__ import annotations

import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from forge_amd import formats as F  # noqa: E402
from forge_amd import ops, step  # noqa: E402

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, FFN, VOCAB, LAYERS, BLOCK = 512, 8, 2, 64, 1024, 2000, 2, 16


def _weight(dtype: int, rows: int, cols: int, g) -> ops.QWeight:
    """Random blocks of a 32-element format, scaled for outputs of unit variance."""
    f = F.fmt(dtype)
    n = rows * cols // f.block_elems
    b = torch.randint(0, 256, (n, f.block_bytes), dtype=torch.uint8, device="cuda", generator=g)
    if dtype == F.Q8_0:
        b[:, 2:] = torch.where(b[:, 2:] == 128, torch.zeros_like(b[:, 2:]), b[:, 2:])
    rms = {F.Q4_0: 4.6, F.Q8_0: 73.0}[dtype]
    d = torch.full((n,), 1.0 / (math.sqrt(cols) * rms), dtype=torch.float16, device="cuda")
    b[:, :2] = d.view(torch.uint8).view(n, 2)
    return ops.QWeight(b.reshape(-1), dtype, rows, cols)


class Model:
    def __init__(self, seed: int = 0, blocks: int = 64):
        g = torch.Generator(device="cuda").manual_seed(seed)
        kv = KV_HEADS * HEAD_DIM
        self.embedding = torch.randn((VOCAB, HIDDEN), device="cuda", generator=g)
        self.layers = [dict(q=_weight(F.Q4_0, HEADS * HEAD_DIM, HIDDEN, g), k=_weight(F.Q4_0, kv, HIDDEN, g),
                            v=_weight(F.Q4_0, kv, HIDDEN, g), o=_weight(F.Q4_0, HIDDEN, HEADS * HEAD_DIM, g),
                            gate=_weight(F.Q4_0, FFN, HIDDEN, g), up=_weight(F.Q4_0, FFN, HIDDEN, g),
                            down=_weight(F.Q8_0, HIDDEN, FFN, g),
                            cache=step.paged_cache(blocks, BLOCK, KV_HEADS, HEAD_DIM))
                       for _ in range(LAYERS)]
        self.head = _weight(F.Q8_0, VOCAB, HIDDEN, g)
        self.norm = torch.ones(HEAD_DIM, device="cuda")
        self.table = step.rope_table(1024, HEAD_DIM)

    def forward(self, tokens, plan, block_table, lengths):
        """Logits [N, VOCAB] of the step's tokens; their keys and values enter the caches."""
        def rms(x):
            return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)

        x = self.embedding[tokens.long()]
        for w in self.layers:
            k, v = w["cache"]
            qkv = ops.fused_qkv(rms(x), w["q"], w["k"], w["v"])
            q = step.qk_norm_rope(qkv, plan.positions, plan.slots, self.table, k, v,
                                  q_weight=self.norm, k_weight=self.norm)
            a = step.tree_attention(q, k, v, block_table, lengths, plan.cu, plan.masks)
            x = x + ops.matmul_transB(a.flatten(1), w["o"])
            x = ops.ffn_down_residual(ops.ffn_up_fused(rms(x), w["gate"], w["up"]), w["down"], x)
        return ops.matmul_transB(rms(x), self.head)


class Requests:
    """Block tables, lengths and free blocks of a batch, on the GPU."""

    def __init__(self, n: int, columns: int = 8, blocks: int = 64):
        self.table = torch.zeros((n, columns), dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
        self.free = torch.arange(blocks, dtype=torch.int32, device="cuda")

    def run(self, model, tokens, new, parents=None):
        """One step's plan and logits (the lengths stay: what is accepted is the caller's)."""
        plan = step.plan_step(self.lengths, new, self.table, self.free, BLOCK, tokens.numel(), parents)
        return plan, model.forward(tokens, plan, self.table, self.lengths)

    def keep(self, plan, new):
        """All of the step's tokens belong to the requests from now on."""
        self.lengths = self.lengths + new
        self.free = self.free[int(plan.info[0]):].contiguous()


def accept(parents, likeliest, draft, root_likeliest):
    """The longest accepted branch of one request's tree, as token numbers: a
    token is accepted where its parent is and the model's likeliest token there is it."""
    best, branch = [], {-1: []}
    for i, p in enumerate(parents):
        want = root_likeliest if p < 0 else likeliest[p]
        if p in branch and draft[i] == want:
            branch[i] = branch[p] + [i]
            best = max(best, branch[i], key=len)
    return best


def main() -> None:
    dev = "cuda"
    model = Model()
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    prompts = [[5, 17, 900, 3, 42], [7] * 19]
    new = ints([len(p) for p in prompts])
    batch = Requests(len(prompts))
    plan, logits = batch.run(model, ints(sum(prompts, [])), new)
    batch.keep(plan, new)
    last = step.token_logprobs(logits[plan.cu[1:].long() - 1], top=3).top_tokens.tolist()
    # a tree for each request: the model's likeliest token, two alternatives, children of the first
    parents = [-1, -1, -1, 0, 0]
    draft = [t + [11 + i, 1200 + i] for i, t in enumerate(last)]
    plan, logits = batch.run(model, ints(sum(draft, [])), ints([5, 5]), parents=ints(parents * 2))
    scores = step.token_logprobs(logits, top=1)  # what the model would say after each drafted token
    for r in range(2):
        rows = scores.top_tokens[5 * r:5 * r + 5, 0].tolist()
        kept = accept(parents, rows, draft[r], last[r][0])
        print(f"request {r}: draft {draft[r]}, accepted {[draft[r][i] for i in kept]}, "
              f"entropies {[round(v, 2) for v in scores.entropy[5 * r:5 * r + 5].tolist()]}")
    # the same tokens branch by branch, as plain chains on a fresh cache
    worst = 0.0
    for branch in ([0], [1], [2], [0, 3], [0, 4]):
        alone = Requests(2)
        fresh = Model()
        p, _ = alone.run(fresh, ints(sum(prompts, [])), new)
        alone.keep(p, new)
        n = ints([len(branch)] * 2)
        _, chain = alone.run(fresh, ints([d[i] for d in draft for i in branch]), n)
        for r in range(2):
            a, b = chain[(r + 1) * len(branch) - 1], logits[5 * r + branch[-1]]
            worst = max(worst, float((a - b).norm() / a.norm()))
    print(f"tree against its branches one by one: rel {worst:.2e}")
    # (cached keys and values are fp16, and batches of other sizes round them differently)
    assert worst < 5e-3


if __name__ == "__main__":
    main()
