"""The serving operators' measured cases: page plan, rotary positions with a
cache write, tree attention over the paged cache, and logit rules.

One verification step of a server that drafts tokens runs them in this order;
each case is one of them at sizes such a step meets. ``run`` computes either
the plain form (elementary torch operations in 32 bits) or, with ``own``, the
calls of ``nert_b200.serving``.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decode step of a busy server: 64 requests, one token each
        dict(name="plan_decode", op="plan", batch=64, lo=1, hi=8000, new_lo=1, new_hi=1, block=16, tree=False),
        # a verification step: trees of 24 to 64 drafted tokens, some requests idle
        dict(name="plan_tree", op="plan", batch=129, lo=0, hi=20000, new_lo=0, new_hi=64, block=32, tree=True),
        # long prompts admitted together, cached a block at a time
        dict(name="plan_prompts", op="plan", batch=40, lo=0, hi=900, new_lo=500, new_hi=33000, block=64, tree=False),
        # one decode step: 64 tokens, grouped heads, three position axes
        dict(name="rope_decode", op="rope", tokens=64, heads=32, kv_heads=8, dim=128, rot=128, sections="16 24 24",
             pairs=False, dtype="bf16", cache=True, block=16, span=8000),
        # a video prompt: time, height and width axes, written to the cache
        dict(name="rope_video", op="rope", tokens=16001, heads=28, kv_heads=4, dim=128, rot=128,
             sections="16 24 24", pairs=False, dtype="bf16", cache=True, block=32, span=4096),
        # ViT-B/16 heads over 32 images of 197 tokens: two axes, adjacent pairs, half of the head, no cache
        dict(name="rope_image", op="rope", tokens=6304, heads=12, kv_heads=12, dim=64, rot=32, sections="8 8",
             pairs=True, dtype="f32", cache=False, block=16, span=224),
        # few requests, one token each: latency counts
        dict(name="attn_decode", op="attn", batch=4, lo=60, hi=2000, new_lo=1, new_hi=1, heads=32, kv_heads=8, dim=128,
             block=16, dtype="bf16"),
        # verification of wide trees over ordinary contexts
        dict(name="attn_tree", op="attn", batch=16, lo=300, hi=6000, new_lo=33, new_hi=64, heads=32, kv_heads=8,
             dim=128, block=16, dtype="bf16"),
        # narrow trees over long contexts, an odd number of heads a group
        dict(name="attn_long", op="attn", batch=8, lo=9000, hi=60000, new_lo=7, new_hi=16, heads=40, kv_heads=8,
             dim=128, block=64, dtype="f16"),
        # ViT-B/16 heads in the framework's own type, every head with its own keys
        dict(name="attn_f32", op="attn", batch=8, lo=100, hi=3000, new_lo=5, new_hi=24, heads=12, kv_heads=12, dim=64,
             block=16, dtype="f32"),
        # a few rows of an odd vocabulary
        dict(name="logits_few", op="logits", requests=3, per=1, vocab=32003, history=700, bias=20, grammar=True,
             dtype="f32"),
        # every drafted token of 24 trees, each with its own grammar state
        dict(name="logits_trees", op="logits", requests=24, per=17, vocab=128000, history=6000, bias=300, grammar=True,
             dtype="bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["plan", "rope", "attn", "attn", "logits"])
    if op == "plan":
        tree = rng.random() < 0.5
        batch = log(1, 300)
        new_hi = rng.randint(1, 96) if tree else log(1, max(1, 600000 // batch))
        return dict(op=op, batch=batch, lo=0, hi=log(10, 30000), new_lo=rng.randint(0, new_hi), new_hi=new_hi,
                    block=rng.choice([8, 16, 24, 32, 64, 128]), tree=tree)
    if op == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([dim, dim, dim // 2])
        kv = rng.choice([1, 2, 4, 8])
        axes = rng.randint(1, 3)
        half = rot // 2
        cut = sorted(rng.randint(0, half) for _ in range(axes - 1))
        sections = " ".join(str(b - a) for a, b in zip([0] + cut, cut + [half]))
        return dict(op=op, tokens=log(1, 12000), heads=kv * rng.choice([1, 3, 4, 7]), kv_heads=kv, dim=dim, rot=rot,
                    sections=sections, pairs=rng.random() < 0.4, dtype=rng.choice(["bf16", "f16", "f32"]),
                    cache=rng.random() < 0.7, block=rng.choice([8, 16, 24, 64]), span=log(100, 30000))
    if op == "attn":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        dim = rng.choice([64, 80, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        batch = log(1, 40)
        hi = log(20, max(40, min(40000, 60_000_000 // (batch * kv * dim))))
        new_hi = rng.choice([1, log(2, 100), log(2, 100)])
        return dict(op=op, batch=batch, lo=0, hi=hi, new_lo=rng.randint(0 if batch > 1 else 1, new_hi), new_hi=new_hi,
                    heads=kv * rng.choice([1, 3, 4, 5, 8]), kv_heads=kv, dim=dim, block=rng.choice([8, 16, 24, 64]),
                    dtype=dtype)
    per = rng.choice([1, 1, rng.randint(2, 20)])
    vocab = log(1000, 200000)
    return dict(op=op, requests=log(1, max(2, min(200, 60_000_000 // (vocab * per)))), per=per, vocab=vocab,
                history=log(1, 20000), bias=rng.choice([0, log(1, 400)]), grammar=rng.random() < 0.6,
                dtype=rng.choice(["f32", "f16", "bf16"]))


# ---- the sizes of a case, which its name and seed do not change ----------------------------------------------------


def _spread(n, lo, hi, shift):
    """n whole numbers over lo..hi, evenly spread, in no order; the ends are among them."""
    u = (np.arange(n) * 0.6180339887498949 + shift) % 1.0
    v = lo + np.floor(u * (hi - lo + 1)).astype(np.int64)
    if n > 1:
        v[0] = hi
        v[1] = lo
    else:
        v[:] = hi
    return v


def _lens(case):
    return _spread(case["batch"], case["lo"], case["hi"], 0.37), _spread(case["batch"], case["new_lo"], case["new_hi"], 0.71)[::-1]


def _tree(n, r):
    """Parents of n drafted tokens: a chain, or two to four children each; every fifth request has two roots."""
    p = (np.arange(n) - 1) // (1 + r % 4)
    p[:1] = -1
    if r % 5 == 4 and n > 1:
        p[1] = -1
    return p


def _visible(n, r):
    """Pairs of a drafted token with itself or an ancestor."""
    depth = np.zeros(n, np.int64)
    for i, p in enumerate(_tree(n, r)):
        depth[i] = 1 if p < 0 else depth[p] + 1
    return int(depth.sum())


def work(case):
    if case["op"] == "plan":
        old, new = _lens(case)
        s = case["block"]
        fresh = int(((old + new + s - 1) // s - (old + s - 1) // s).sum())
        t = int(new.sum())
        words = (case["new_hi"] + 31) // 32 if case["tree"] else 0
        n = 2 * case["batch"] + 2 * fresh + t * (2 + words + (1 if case["tree"] else 0)) + 3 * case["batch"] + 2
        return {"bytes": 4 * n, "flops": 2 * t}
    if case["op"] == "rope":
        t, e, d = case["tokens"], BYTES[case["dtype"]], case["dim"]
        rows = case["heads"] + case["kv_heads"] * (2 if case["cache"] else 1)
        table = min(t, case["span"]) * case["rot"] * 4
        ints = t * 4 * (len(case["sections"].split()) + (1 if case["cache"] else 0))
        return {"bytes": 2 * t * rows * d * e + table + ints,
                "flops": 3 * t * (case["heads"] + case["kv_heads"]) * case["rot"]}
    if case["op"] == "attn":
        old, new = _lens(case)
        e, d = BYTES[case["dtype"]], case["dim"]
        t = int(new.sum())
        pairs = int((old * new).sum()) + sum(_visible(int(n), r) for r, n in enumerate(new))
        words = (case["new_hi"] + 31) // 32
        live = old[new > 0] + new[new > 0]
        cache = int(live.sum()) * case["kv_heads"] * d * 2 * e
        table = int(((live + case["block"] - 1) // case["block"]).sum()) * 4
        return {"bytes": cache + 2 * t * case["heads"] * d * e + t * words * 4 + t * case["heads"] * 4 + table,
                "flops": 4 * d * case["heads"] * pairs}
    rows, v = case["requests"] * case["per"], case["vocab"]
    ids = sum(int(x.sum()) for x in _history(case))
    mask = rows * ((v + 31) // 32) * 4 if case["grammar"] else 0
    return {"bytes": rows * v * (BYTES[case["dtype"]] + 4) + ids * 4 + case["requests"] * case["bias"] * 8 + mask,
            "flops": rows * v}


def _history(case):
    """Lengths of the prompts and of the answers so far."""
    return (_spread(case["requests"], case["history"] // 8, case["history"], 0.2),
            _spread(case["requests"], 0, max(1, case["history"] // 3), 0.55))


# ---- inputs -----------------------------------------------------------------------------------------------------


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def _pages(rng, old, new, block, spare):
    """A pool's blocks in random order: the block table of what is cached, and the free blocks after them."""
    have = (old + block - 1) // block
    want = (old + new + block - 1) // block
    pool = rng.permutation(int(want.sum()) + spare)
    table = np.full((len(old), max(1, int(want.max()))), -1, np.int64)
    at = 0
    for r, h in enumerate(have):
        table[r, :h] = pool[at:at + h]
        at += h
    return table, pool[at:], want, len(pool)


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype="f32", scale=1.0):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=DTYPES[dtype])
        return x if scale == 1.0 else x.mul_(scale)

    op = case["op"]
    if op in ("plan", "attn"):
        old, new = _lens(case)
        order = rng.permutation(case["batch"])
        old, new = old[order], new[order]
        trees = [_tree(int(n), int(r)) for r, n in zip(order, new)]
        parents = np.concatenate(trees + [np.zeros(0, np.int64)])
        words = (case["new_hi"] + 31) // 32
    if op == "plan":
        table, free, _, _ = _pages(rng, old, new, case["block"], 100)
        wide = int(((old + new + case["block"] - 1) // case["block"]).max()) + 3
        full = np.full((case["batch"], wide), -1, np.int64)
        full[:, :table.shape[1]] = table
        return dict(case=case, seq_lens=_i32(old), new_lens=_i32(new), table=_i32(full), free=_i32(free[5:]),
                    head=_i32([7]), tokens=int(new.sum()), words=words if case["tree"] else 0,
                    parents=_i32(parents) if case["tree"] else None)
    if op == "rope":
        t, h, kv, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        qkv = normal(t, (h + 2 * kv) * d, dtype=case["dtype"])
        q, k, v = qkv.split([h * d, kv * d, kv * d], dim=1)
        half = case["rot"] // 2
        freq = 10000.0 ** (-np.arange(half) / half)
        angle = np.arange(case["span"])[:, None] * freq[None, :]
        table = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).cuda()
        sections = [int(n) for n in case["sections"].split()]
        axis_of = [a for a, n in enumerate(sections) for _ in range(n)]
        pos = rng.integers(0, case["span"], (len(sections), t))
        state = dict(case=case, q=q.view(t, h, d), k=k.view(t, kv, d), v=v.view(t, kv, d), table=table, pos=_i32(pos),
                     axis_of=tuple(axis_of))
        if case["cache"]:
            blocks = (t + case["block"] - 1) // case["block"] + 9
            slots = rng.permutation(blocks)[:, None] * case["block"] + np.arange(case["block"])[None, :]
            state["slots"] = _i32(slots.reshape(-1)[:t])
            state["k_cache"] = normal(blocks, case["block"], kv, d, dtype=case["dtype"])
            state["v_cache"] = normal(blocks, case["block"], kv, d, dtype=case["dtype"])
        return state
    if op == "attn":
        d, h, kv, s = case["dim"], case["heads"], case["kv_heads"], case["block"]
        table, free, want, blocks = _pages(rng, old, new, s, 20)
        have = (old + s - 1) // s
        at = 0
        for r, (a, b) in enumerate(zip(have, want)):
            table[r, a:b] = free[at:at + b - a]
            at += b - a
        rows = [np.eye(int(n), dtype=bool) for n in new]
        for m, p in zip(rows, trees):
            for i, j in enumerate(p):
                if j >= 0:
                    m[i] |= m[j]
        mask = np.zeros((len(parents), words * 32), bool)
        at = 0
        for m in rows:
            mask[at:at + len(m), :len(m)] = m
            at += len(m)
        bits = np.packbits(mask, axis=1, bitorder="little").view(np.uint32).view(np.int32).reshape(len(parents), words)
        return dict(case=case, q=normal(int(new.sum()), h, d, dtype=case["dtype"], scale=1.5),
                    k_cache=normal(blocks, s, kv, d, dtype=case["dtype"]),
                    v_cache=normal(blocks, s, kv, d, dtype=case["dtype"]), table=_i32(table),
                    total=_i32(old + new), offsets=_i32(_offsets(new)), mask=_i32(bits), scale=1.0 / math.sqrt(d),
                    max_new=case["new_hi"], longest=int((old + new).max()))
    v, req, per = case["vocab"], case["requests"], case["per"]
    prompt, answer = _history(case)
    order = rng.permutation(req)
    prompt, answer = prompt[order], answer[order]

    def words_of(n):  # tokens of a text: few common ones, many rare ones
        return np.minimum((v * rng.random(n) ** 3).astype(np.int64), v - 1)

    state = dict(case=case, logits=normal(req * per, v, dtype=case["dtype"], scale=3.0),
                 prompt_ids=_i32(words_of(int(prompt.sum()))), prompt_offsets=_i32(_offsets(prompt)),
                 output_ids=_i32(words_of(int(answer.sum()))), output_offsets=_i32(_offsets(answer)),
                 row_request=_i32(np.repeat(np.arange(req), per)),
                 repetition=torch.from_numpy(rng.uniform(1.0, 1.4, req).astype(np.float32)).cuda(),
                 presence=torch.from_numpy(rng.uniform(-0.2, 0.8, req).astype(np.float32)).cuda(),
                 frequency=torch.from_numpy(rng.uniform(0.0, 0.5, req).astype(np.float32)).cuda())
    if case["bias"]:
        n = min(case["bias"], v)
        ids = np.concatenate([rng.choice(v, n, replace=False) for _ in range(req)])
        state["bias_ids"] = _i32(ids)
        state["bias_values"] = torch.from_numpy(rng.normal(0, 4, len(ids)).astype(np.float32)).cuda()
        state["bias_offsets"] = _i32(np.arange(req + 1) * n)
    if case["grammar"]:
        w = (v + 31) // 32
        mask = torch.randint(-2**31, 2**31, (req * per, w), generator=gen, device="cuda", dtype=torch.int32)
        state["grammar"] = mask
        state["grammar_rows"] = _i32(np.where(np.arange(req * per) % 7 == 6, -1, np.arange(req * per)))
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------


def _bits(words, n):
    """[..., W] whole words -> [..., n] truth values, bit j of word w at 32 w + j."""
    b = (words.unsqueeze(-1) >> torch.arange(32, device=words.device, dtype=torch.int32)) & 1
    return b.flatten(-2)[..., :n] != 0


def _plain_plan(s):
    c, size = s["case"], s["case"]["block"]
    old, new = s["seq_lens"].long(), s["new_lens"].long()
    have, want = (old + size - 1) // size, (old + new + size - 1) // size
    fresh = want - have
    first = fresh.cumsum(0) - fresh + s["head"].long()
    col = torch.arange(s["table"].shape[1], device="cuda")
    is_new = (col >= have[:, None]) & (col < want[:, None])
    take = (first[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    s["table"].copy_(torch.where(is_new, s["free"][take], s["table"]))
    ends = new.cumsum(0)
    offsets = torch.cat([ends.new_zeros(1), ends])
    t = torch.arange(s["tokens"], device="cuda")
    req = torch.searchsorted(ends, t, right=True)
    i = t - offsets[req]
    p = old[req] + i
    slots = s["table"][req, p // size] * size + (p % size).int()
    head = (s["head"].long() + fresh.sum()).int()
    if not c["tree"]:
        return (old + new).int(), offsets.int(), slots, p.int(), s["table"], head
    n = s["words"] * 32
    up = s["parents"].long()
    reach = torch.zeros(c["batch"], n, n, device="cuda")
    reach[req, i, i] = 1.0
    step = torch.zeros(c["batch"], n, n, device="cuda")
    step[req, i, up.clamp(min=0)] = (up >= 0).float()
    for _ in range((n - 1).bit_length()):  # ancestors at most 1, 2, 4, ... steps away
        reach = ((reach + step @ reach) > 0).float()
        step = step @ step
    seen = reach[req, i] > 0
    depth = seen.sum(1) - 1
    weight = torch.ones(32, device="cuda", dtype=torch.int64) << torch.arange(32, device="cuda")
    words = (seen.view(-1, s["words"], 32) * weight).sum(-1)
    mask = torch.where(words >= 2**31, words - 2**32, words).int()
    return (old + new).int(), offsets.int(), slots, (old[req] + depth).int(), s["table"], head, mask


def _plain_rope(s):
    c = s["case"]
    half = c["rot"] // 2
    axis = torch.tensor(s["axis_of"], device="cuda")
    row = s["pos"].long()[axis].t()  # [tokens, half]: each frequency's position
    f = torch.arange(half, device="cuda")
    cos, sin = s["table"][row, f].unsqueeze(1), s["table"][row, half + f].unsqueeze(1)

    def turn(x):
        y = x.float().clone()
        a, b = (y[..., 0:c["rot"]:2], y[..., 1:c["rot"]:2]) if c["pairs"] else (y[..., :half], y[..., half:c["rot"]])
        a0, b0 = a.clone(), b.clone()
        a.copy_(a0 * cos - b0 * sin)
        b.copy_(b0 * cos + a0 * sin)
        return y.to(x.dtype)

    q, k = turn(s["q"]), turn(s["k"])
    if not c["cache"]:
        return q, k
    at = s["slots"].long()
    s["k_cache"].view(-1, c["kv_heads"], c["dim"])[at] = k
    s["v_cache"].view(-1, c["kv_heads"], c["dim"])[at] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_attn(s):
    c = s["case"]
    group, d, size, b = c["heads"] // c["kv_heads"], c["dim"], c["block"], c["batch"]
    total, start = s["total"].long(), s["offsets"].long()
    new = start[1:] - start[:-1]
    at = torch.arange(s["longest"], device="cuda")
    page = s["table"].long().clamp(min=0)[:, at // size]  # [b, longest]
    k = s["k_cache"][page, at % size].permute(0, 2, 3, 1).float()  # [b, kv, d, longest]
    v = s["v_cache"][page, at % size].permute(0, 2, 1, 3).float()  # [b, kv, longest, d]
    n = s["max_new"]
    i = torch.arange(n, device="cuda")
    token = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)  # [b, n]
    q = s["q"][token].float().view(b, n, c["kv_heads"], group, d).permute(0, 2, 1, 3, 4).reshape(b, c["kv_heads"], n * group, d)
    tail = at - (total - new)[:, None]  # [b, longest]: index among the new tokens
    own_bits = _bits(s["mask"], 32 * s["mask"].shape[1])[token]  # [b, n, 32 W]
    drafted = own_bits.gather(2, tail.clamp(0, own_bits.shape[2] - 1)[:, None, :].expand(b, n, -1))
    see = ((tail < 0)[:, None, :] | drafted & (tail < new[:, None])[:, None, :]) & (at < total[:, None])[:, None, :]
    score = (q @ k).mul_(s["scale"]).view(b, c["kv_heads"], n, group, -1)
    score.masked_fill_(~see[:, None, :, None, :], -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    z = p.sum(-1, keepdim=True)
    o = (p.view(b, c["kv_heads"], n * group, -1) @ v).view(b, c["kv_heads"], n, group, d) / z
    lse = (top + z.log()).squeeze(-1)
    live = i < new[:, None]
    o = o.permute(0, 2, 1, 3, 4).reshape(b, n, c["heads"], d)[live]
    return o.to(s["q"].dtype), lse.permute(0, 2, 1, 3).reshape(b, n, c["heads"])[live]


def _plain_logits(s):
    c = s["case"]
    v, req = c["vocab"], c["requests"]

    def owner(offsets, n):
        return torch.searchsorted(offsets[1:].long(), torch.arange(n, device="cuda"), right=True)

    ids = s["output_ids"].long()
    count = torch.zeros(req, v, device="cuda")
    count.index_put_((owner(s["output_offsets"], ids.numel()), ids), torch.ones(1, device="cuda"), accumulate=True)
    seen = count > 0
    ids = s["prompt_ids"].long()
    seen[owner(s["prompt_offsets"], ids.numel()), ids] = True
    less = s["frequency"][:, None] * count + s["presence"][:, None] * (count > 0).float()
    more = torch.zeros(req, v, device="cuda")
    if c["bias"]:
        ids = s["bias_ids"].long()
        more[owner(s["bias_offsets"], ids.numel()), ids] = s["bias_values"]
    r = s["row_request"].long()
    x = s["logits"].float()
    rep = s["repetition"][r][:, None]
    x = torch.where(seen[r], torch.where(x > 0, x / rep, x * rep), x) - less[r] + more[r]
    if c["grammar"]:
        g = s["grammar_rows"].long()
        allowed = _bits(s["grammar"], v)[g.clamp(min=0)] | (g < 0)[:, None]
        x = x.masked_fill(~allowed, -math.inf)
    return x


PLAIN = {"plan": _plain_plan, "rope": _plain_rope, "attn": _plain_attn, "logits": _plain_logits}


# ---- the framework's calls ----------------------------------------------------------------------------------------


def _own(s):
    from nert_b200 import serving

    c = s["case"]
    if c["op"] == "plan":
        p = serving.page_plan(s["seq_lens"], s["new_lens"], s["table"], s["free"], c["block"], s["tokens"],
                              parents=s["parents"], mask_words=s["words"], free_head=s["head"])
        out = (p.seq_lens, p.token_offsets, p.slots, p.positions, s["table"], p.free_head)
        return out + (p.tree_mask,) if c["tree"] else out
    if c["op"] == "rope":
        if not c["cache"]:
            return serving.rope_append(s["q"], s["k"], None, s["table"], s["pos"], axis_of=s["axis_of"],
                                       interleaved=c["pairs"])
        q, _ = serving.rope_append(s["q"], s["k"], s["v"], s["table"], s["pos"], axis_of=s["axis_of"],
                                   interleaved=c["pairs"], slots=s["slots"], k_cache=s["k_cache"],
                                   v_cache=s["v_cache"])
        return q, s["k_cache"], s["v_cache"]
    if c["op"] == "attn":
        return serving.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["total"], s["offsets"],
                                      tree_mask=s["mask"], max_new=s["max_new"], scale=s["scale"], return_lse=True)
    return serving.logits_process(
        s["logits"], prompt=(s["prompt_ids"], s["prompt_offsets"]), output=(s["output_ids"], s["output_offsets"]),
        row_request=s["row_request"], repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
        bias=(s["bias_ids"], s["bias_values"], s["bias_offsets"]) if c["bias"] else None,
        grammar=(s["grammar"], s["grammar_rows"]) if c["grammar"] else None, out_dtype=torch.float32)


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        half = case["rot"] // 2
        table, pos = s["table"].double(), s["pos"].long()
        first = [2 * f if case["pairs"] else f for f in range(half)]
        second = [2 * f + 1 if case["pairs"] else half + f for f in range(half)]

        def turned(x):
            y = x.double()
            z = torch.complex(y[..., first], y[..., second])
            w = torch.complex(torch.stack([table[pos[a], f] for f, a in enumerate(s["axis_of"])], -1),
                              torch.stack([table[pos[a], half + f] for f, a in enumerate(s["axis_of"])], -1))
            z = z * w[:, None, :]
            y[..., first] = z.real
            y[..., second] = z.imag
            return y

        q, k = turned(s["q"]), turned(s["k"])
        if not case["cache"]:
            return q, k
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        at = s["slots"].long()
        kc[at // case["block"], at % case["block"]] = k
        vc[at // case["block"], at % case["block"]] = s["v"].double()
        return q, kc, vc
    if case["op"] == "attn":
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        offsets, total, mask = s["offsets"].tolist(), s["total"].tolist(), s["mask"].cpu().numpy().view(np.uint32)
        for r, n_all in enumerate(total):
            a, b = offsets[r], offsets[r + 1]
            if a == b:
                continue
            old = n_all - (b - a)
            see = np.ones((b - a, n_all), bool)
            see[:, old:] = np.unpackbits(mask[a:b].view(np.uint8), axis=1, bitorder="little")[:, :b - a]
            see = torch.from_numpy(see).cuda()
            pages = s["table"][r, :(n_all + case["block"] - 1) // case["block"]].long()
            for h in range(case["kv_heads"]):
                k = s["k_cache"][pages, :, h].reshape(-1, case["dim"])[:n_all].double()
                v = s["v_cache"][pages, :, h].reshape(-1, case["dim"])[:n_all].double()
                for g in range(h * group, (h + 1) * group):
                    x = s["q"][a:b, g].double() @ k.T * s["scale"]
                    x[~see] = -math.inf
                    lse[a:b, g] = torch.logsumexp(x, -1)
                    out[a:b, g] = torch.softmax(x, -1) @ v
        return out, lse
    if case["op"] == "logits":
        x = s["logits"].double()
        prompt, answer, bias = (s[n].tolist() if n in s else None for n in ("prompt_offsets", "output_offsets", "bias_offsets"))
        for r in range(case["requests"]):
            count = torch.bincount(s["output_ids"][answer[r]:answer[r + 1]].long(), minlength=case["vocab"])
            seen = (count > 0) | (torch.bincount(s["prompt_ids"][prompt[r]:prompt[r + 1]].long(), minlength=case["vocab"]) > 0)
            y = x[r * case["per"]:(r + 1) * case["per"]]
            rep = s["repetition"][r].double()
            y[:, seen] = torch.where(y[:, seen] > 0, y[:, seen] / rep, y[:, seen] * rep)
            y -= s["frequency"][r].double() * count + s["presence"][r].double() * (count > 0)
            if bias is not None:
                y[:, s["bias_ids"][bias[r]:bias[r + 1]].long()] += s["bias_values"][bias[r]:bias[r + 1]].double()
        if case["grammar"]:
            bits = np.unpackbits(s["grammar"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :case["vocab"]]
            rows = s["grammar_rows"].tolist()
            keep = torch.from_numpy(bits != 0).cuda()
            for r, m in enumerate(rows):
                if m >= 0:
                    x[r, ~keep[m]] = -math.inf
        return x
    old, new = s["seq_lens"].cpu().numpy().astype(np.int64), s["new_lens"].cpu().numpy().astype(np.int64)
    table, free, head, size = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy(), int(s["head"][0]), case["block"]
    up = s["parents"].cpu().numpy() if case["tree"] else None
    slots, places, masks = [], [], []
    for r in range(case["batch"]):
        for j in range(-(-old[r] // size), -(-(old[r] + new[r]) // size)):
            table[r, j] = free[head]
            head += 1
        p = old[r] + np.arange(new[r])
        slots.append(table[r, p // size].astype(np.int64) * size + p % size)
        if up is None:
            places.append(p)
            continue
        at = sum(len(x) for x in places)
        depth, seen = np.zeros(new[r], np.int64), np.zeros((new[r], 32 * s["words"]), np.uint8)
        for i in range(new[r]):
            j = up[at + i]
            if j >= 0:
                depth[i] = depth[j] + 1
                seen[i] = seen[j]
            seen[i, i] = 1
        places.append(old[r] + depth)
        masks.append(np.packbits(seen, axis=1, bitorder="little").view(np.int32).reshape(new[r], s["words"]))
    out = (_i32(old + new), _i32(_offsets(new)), _i32(np.concatenate(slots)), _i32(np.concatenate(places)), _i32(table), _i32([head]))
    return out + (_i32(np.concatenate(masks)),) if case["tree"] else out
