"""Drafted tokens verified over a paged cache, with the rows of this library.

A small decoder (random weights, float32) serves a few requests at once. Each
step takes a tree of drafted tokens a request and runs, in one pass over all of
them: the page plan, then for each layer LayerNormalization, the q/k/v Gemm,
rotary positions with the cache write, tree attention and the MLP, and at the
end the logit rules and TopK. The longest drafted path that the model agrees
with is kept, and one token more.

    python examples/verify_drafts.py [--steps N]

All rows run on torch's current stream, through the context that the serving
rows use; the host waits once a step, for the tokens.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from nert_b200 import _lib, serving  # noqa: E402
from nert_b200._lib import check, lib  # noqa: E402


class Linear:
    """A weight [n, k] packed once for the Gemm row."""

    def __init__(self, n: int, k: int, gen, scale: float | None = None):
        w = torch.randn(n, k, device="cuda", generator=gen) * (k**-0.5 if scale is None else scale)
        size = (_lib.ctypes.c_int64)()
        check(lib().nb2_gemm_packed_size(n, k, _lib.ctypes.byref(size)))
        self.n, self.k, self.weight = n, k, w
        self.packed = torch.empty(size.value, device="cuda", dtype=torch.uint8)
        check(lib().nb2_gemm_pack(serving.context(), w.data_ptr(), n, k, 1, self.packed.data_ptr()))

    def __call__(self, x, residual=None, act=_lib.ACT_NONE):
        y = torch.empty(x.shape[0], self.n, device="cuda")
        check(lib().nb2_gemm_run_packed(serving.context(), x.data_ptr(), self.packed.data_ptr(),
                                        None if residual is None else residual.data_ptr(),
                                        0 if residual is None else 2, y.data_ptr(), x.shape[0], self.n, self.k, 0, 1.0,
                                        1.0, act))
        return y


class Decoder:
    def __init__(self, batch: int, layers=2, heads=8, kv_heads=2, dim=64, vocab=1000, blocks=256, block=16, length=1024,
                 seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.batch, self.heads, self.kv, self.dim, self.vocab, self.block = batch, heads, kv_heads, dim, vocab, block
        self.hidden = heads * dim
        self.embed = torch.randn(vocab, self.hidden, device="cuda", generator=gen)
        self.layers = [dict(qkv=Linear((heads + 2 * kv_heads) * dim, self.hidden, gen), o=Linear(self.hidden, self.hidden, gen),
                            up=Linear(4 * self.hidden, self.hidden, gen), down=Linear(self.hidden, 4 * self.hidden, gen))
                       for _ in range(layers)]
        self.head = Linear(vocab, self.hidden, gen)
        self.one = torch.ones(self.hidden, device="cuda")
        angle = torch.arange(length, device="cuda")[:, None] * 10000.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2))
        self.rope = torch.cat([angle.cos(), angle.sin()], 1).contiguous()
        shape = (layers, blocks, block, kv_heads, dim)
        self.k, self.v = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
        self.table = torch.full((batch, length // block), -1, device="cuda", dtype=torch.int32)
        self.blocks = blocks
        self.lens = [0] * batch  # cached tokens

    def norm(self, x):
        y = torch.empty_like(x)
        check(lib().nb2_layernorm(serving.context(), x.data_ptr(), self.one.data_ptr(), None, y.data_ptr(), None, None,
                                  x.shape[0], self.hidden, 1e-5))
        return y

    def forward(self, tokens: list[list[int]], parents: list[list[int]] | None = None):
        """Logits of every new token (rows in order of the requests), and the plan. With ``parents`` the new tokens of
        a request are a tree; nothing is committed: ``commit`` does."""
        new = [len(t) for t in tokens]
        flat = [t for r in tokens for t in r]
        i32 = lambda x: torch.tensor(x, device="cuda", dtype=torch.int32)  # noqa: E731
        # the pool's free blocks: what no committed token lies in
        table = self.table.tolist()
        used = {b for r, n in enumerate(self.lens) for b in table[r][:-(-n // self.block)]}
        free = i32([b for b in range(self.blocks) if b not in used])
        plan = serving.page_plan(i32(self.lens), i32(new), self.table, free, self.block, len(flat),
                                 parents=None if parents is None else i32([p for r in parents for p in r]),
                                 mask_words=0 if parents is None else -(-max(new) // 32))
        ids = torch.tensor(flat, device="cuda", dtype=torch.int64)
        x = torch.empty(len(flat), self.hidden, device="cuda")
        check(lib().nb2_gather(serving.context(), self.embed.data_ptr(), ids.data_ptr(), x.data_ptr(), 1, self.vocab,
                               self.hidden, len(flat), 4))
        h, kv, d = self.heads, self.kv, self.dim
        for n, w in enumerate(self.layers):
            qkv = w["qkv"](self.norm(x))
            q, k, v = (t.view(len(flat), -1, d) for t in qkv.split([h * d, kv * d, kv * d], dim=1))
            q, _ = serving.rope_append(q, k, v, self.rope, plan.positions, slots=plan.slots, k_cache=self.k[n],
                                       v_cache=self.v[n])
            a = serving.tree_attention(q, self.k[n], self.v[n], self.table, plan.seq_lens, plan.token_offsets,
                                       tree_mask=plan.tree_mask, max_new=max(new))
            x = w["o"](a.view(len(flat), self.hidden), residual=x)
            x = w["down"](w["up"](self.norm(x), act=_lib.ACT_SILU), residual=x)
        return self.head(self.norm(x)), plan

    def commit(self, plan, kept: list[list[int]]):
        """Keeps these new tokens (indices, a path from the root) of each request: their keys and values move to the
        places after the cached ones. A kept token's position is the place it moves to."""
        starts, slots = plan.token_offsets.tolist(), plan.slots.tolist()
        src = [slots[starts[r] + i] for r, path in enumerate(kept) for i in path]
        dst = [slots[starts[r] + j] for r, path in enumerate(kept) for j in range(len(path))]
        if src != dst:
            a, b = torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda")
            for c in (self.k, self.v):
                flat = c.view(c.shape[0], -1, self.kv, self.dim)
                flat[:, b] = flat[:, a]
        self.lens = [n + len(path) for n, path in zip(self.lens, kept)]

    def pick(self, logits, requests: list[int], prompts, outputs, rules):
        """Most likely token of every row after the request's rules (logit rules, then TopK)."""
        def ragged(lists):
            ends = torch.tensor([len(x) for x in lists]).cumsum(0)
            return (torch.tensor([t for x in lists for t in x], device="cuda", dtype=torch.int32),
                    torch.cat([torch.zeros(1, dtype=torch.int64), ends]).to("cuda", torch.int32))

        rows = logits.shape[0]
        serving.logits_process(logits, prompt=ragged(prompts), output=ragged(outputs),
                               row_request=torch.tensor(requests, device="cuda", dtype=torch.int32), out=logits, **rules)
        values = torch.empty(rows, 1, device="cuda")
        best = torch.empty(rows, 1, device="cuda", dtype=torch.int64)
        check(lib().nb2_topk(serving.context(), logits.data_ptr(), values.data_ptr(), best.data_ptr(), rows, self.vocab, 1))
        serving.synchronize()
        return best.flatten().tolist()


def draft(model, rng, last: list[int], depth: int, extra: int) -> tuple[list[list[int]], list[list[int]]]:
    """A tree a request after the committed text, rooted at its last token: the model's own most likely
    continuation without the rules (a real drafter is a smaller model), and `extra` random side branches."""
    tokens, parents = [[t] for t in last], [[-1] for _ in last]
    for _ in range(depth):
        logits, plan = model.forward(tokens)
        ends = plan.token_offsets[1:].long() - 1
        for r, t in enumerate(logits[ends].argmax(1).tolist()):
            parents[r].append(len(tokens[r]) - 1)
            tokens[r].append(t)
    for r in range(len(last)):
        for _ in range(int(rng.integers(extra + 1))):
            parents[r].append(int(rng.integers(len(tokens[r]))))
            tokens[r].append(int(rng.integers(model.vocab)))
    return tokens, parents


def main():
    import numpy as np

    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=6)
    steps = ap.parse_args().steps
    rng = np.random.default_rng(0)
    batch = 3
    model = Decoder(batch)
    prompts = [rng.integers(0, model.vocab, n).tolist() for n in (37, 5, 120)]
    outputs: list[list[int]] = [[] for _ in prompts]
    rules = dict(repetition=torch.full((batch,), 1.1, device="cuda"), presence=torch.zeros(batch, device="cuda"),
                 frequency=torch.full((batch,), 0.1, device="cuda"))
    # the prompts, all but their last token (the root of the first tree)
    _, plan = model.forward([p[:-1] for p in prompts])
    model.commit(plan, [list(range(len(p) - 1)) for p in prompts])
    last = [p[-1] for p in prompts]
    for step in range(steps):
        tokens, parents = draft(model, rng, last, depth=3, extra=6)
        logits, plan = model.forward(tokens, parents)
        rows = [r for r, t in enumerate(tokens) for _ in t]
        best = model.pick(logits, rows, prompts, outputs, rules)
        kept, at = [], 0
        for r in range(batch):
            path, i = [0], 0
            while True:  # down the tree as long as a drafted token is the one the model picks
                want = best[at + i]
                i = next((j for j, p in enumerate(parents[r]) if p == i and tokens[r][j] == want), None)
                if i is None:
                    break
                path.append(i)
            outputs[r] += [tokens[r][j] for j in path[1:]] + [want]
            last[r] = want
            kept.append(path)
            at += len(tokens[r])
        model.commit(plan, kept)
        print(f"step {step}: drafted {[len(t) - 1 for t in tokens]}, kept {[len(p) - 1 for p in kept]}, cached {model.lens}")
    for r, o in enumerate(outputs):
        print(f"request {r}: {o}")


if __name__ == "__main__":
    main()
