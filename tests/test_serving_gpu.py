"""The serving rows (page plan, rotary positions with the cache write, tree
attention, logit rules) on the GPU against plain implementations in 64 bits.

Tolerances are bounds, not fits. With u the unit roundoff of the stored type
(2^-24, 2^-11, 2^-8 for float32, float16, bfloat16): a result rounded once is
off by at most u times itself; a product or sum held in float32 by 2^-24 times
the sum of its terms' magnitudes for each operation. Each check below says how
many operations it allows."""

import math

import numpy as np
import pytest
import torch

from nert_b200 import _lib, serving

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
SMALLEST = {"f32": 2.0**-126, "f16": 2.0**-24, "bf16": 2.0**-126}  # absolute rounding of the type near zero


def i32(x):
    return torch.tensor(np.asarray(x, np.int32), device="cuda")


def device_error(fn):
    """fn's launches record a device error, and the context stays usable."""
    serving.synchronize()
    fn()
    with pytest.raises(_lib.NB2Error) as e:
        serving.synchronize()
    assert e.value.status == _lib.ERR_DEVICE
    serving.synchronize()


def np64(t):
    return t.detach().to(torch.float64).cpu().numpy()


# ---- page plan --------------------------------------------------------------------------------------------------


def plan_ref(old, new, table, free, head, block, tokens, parents, words):
    table = table.copy()
    total, offsets = old + new, np.concatenate([[0], np.cumsum(new)])
    slots, pos = np.full(tokens, -1), np.zeros(tokens, int)
    mask = np.zeros((tokens, max(words, 1) * 32), bool)
    for r in range(len(old)):
        for j in range(-(-old[r] // block), -(-(old[r] + new[r]) // block)):
            table[r, j] = free[head]
            head += 1
        for i in range(new[r]):
            t, p = offsets[r] + i, old[r] + i
            slots[t] = table[r, p // block] * block + p % block
            pos[t] = p
            if parents is not None:
                chain, j = [], i
                while j >= 0:
                    chain.append(j)
                    j = parents[t - i + j]
                mask[t, chain] = True
                pos[t] = old[r] + len(chain) - 1
    bits = np.packbits(mask, axis=1, bitorder="little").view(np.int32)[:, :words]
    return total, offsets, slots, pos, table, head, bits


def tree_parents(rng, n, kind):
    if kind == "chain":
        return np.arange(n) - 1
    if kind == "star":
        return np.full(n, -1)
    return np.array([rng.integers(-1, i) if i else -1 for i in range(n)], int)


PLANS = [
    # batch, old range, new range, block, padding tokens, tree kind
    (1, (0, 0), (1, 1), 16, 0, None), (1, (15, 15), (2, 2), 16, 3, None), (64, (0, 500), (1, 1), 16, 0, None),
    (37, (0, 90), (0, 40), 7, 11, None), (5, (0, 3), (900, 3000), 64, 1, None), (300, (0, 100), (0, 3), 1, 0, None),
    (9, (0, 70), (0, 64), 8, 5, "random"), (4, (0, 70), (33, 33), 24, 0, "chain"), (3, (5, 9), (96, 130), 16, 0, "star"),
    (1, (1000, 1000), (1024, 1024), 32, 0, "chain"), (2, (3, 8), (1, 1), 16, 2, "random"), (3, (0, 9), (0, 0), 4, 6, None),
    (1500, (0, 40), (0, 5), 4, 0, "random"), (8192, (0, 40), (0, 2), 16, 0, None),
]


@pytest.mark.parametrize("batch,olds,news,block,pad,tree", PLANS)
def test_page_plan(cuda, batch, olds, news, block, pad, tree):
    rng = np.random.default_rng(batch + block)
    old, new = rng.integers(olds[0], olds[1] + 1, batch), rng.integers(news[0], news[1] + 1, batch)
    have, want = -(-old // block), -(-(old + new) // block)
    pool = rng.permutation(int(want.sum()) + 5)
    table = np.full((batch, int(want.max()) + 2), -7)
    at = 0
    for r in range(batch):
        table[r, :have[r]] = pool[at:at + have[r]]
        at += have[r]
    free, head = np.concatenate([[-1, -1], pool[at:]]), 2
    tokens = int(new.sum()) + pad
    words = -(-int(news[1]) // 32) if tree else 0
    parents = None
    if tree:
        parents = np.concatenate([tree_parents(rng, n, tree) for n in new] + [np.zeros(pad)]).astype(int)
    dt = i32(table)
    p = serving.page_plan(i32(old), i32(new), dt, i32(free), block, tokens, parents=None if parents is None else i32(parents),
                          mask_words=words, free_head=i32([head]))
    serving.synchronize()
    total, offsets, slots, pos, table, head, bits = plan_ref(old, new, table, free, head, block, tokens, parents, words)
    for got, want_ in ((p.seq_lens, total), (p.token_offsets, offsets), (p.slots, slots), (p.positions, pos), (dt, table),
                       (p.free_head, [head])):
        assert np.array_equal(got.cpu().numpy(), want_)
    if tree:
        assert np.array_equal(p.tree_mask.cpu().numpy(), bits)


def test_page_plan_errors_on_the_device(cuda):
    def plan(old, new, free=8, cols=4, tokens=8, **kw):
        return serving.page_plan(i32(old), i32(new), i32(np.zeros((len(old), cols))), i32(np.arange(free)), 4, tokens, **kw)

    device_error(lambda: plan([-1], [2]))
    device_error(lambda: plan([1], [-2]))
    device_error(lambda: plan([0, 0], [5, 4]))  # nine tokens in outputs of eight
    device_error(lambda: plan([0], [8], free=1))  # one free block for two
    device_error(lambda: plan([0], [8], cols=1))  # a table row of one block
    device_error(lambda: plan([0], [3], parents=i32([0, -1, -1] + [-1] * 5), mask_words=1))  # its own parent
    device_error(lambda: plan([0], [40], free=20, cols=20, tokens=40, parents=i32(np.arange(40) - 1), mask_words=1))
    out = plan([0], [8], free=1)
    assert out.slots.tolist() == [0, 1, 2, 3, -1, -1, -1, -1]
    with pytest.raises(_lib.NB2Error):
        serving.synchronize()


# ---- rotary positions and the cache write ------------------------------------------------------------------------


def rope_ref(x, table, pos, axis_of, interleaved, rot):
    """(turned, sum of the magnitudes of each element's two products)"""
    half = rot // 2
    y, big = x.copy(), np.abs(x)
    for f in range(half):
        a, b = (2 * f, 2 * f + 1) if interleaved else (f, half + f)
        c, s = table[pos[axis_of[f]], f][:, None], table[pos[axis_of[f]], half + f][:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
        big[..., a] = big[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, big


ROPES = [
    # tokens, q heads, kv heads, dim, rot, sections, interleaved, layout of the cache (None: no cache)
    (1, 1, 1, 2, 2, (1,), False, None), (1, 32, 8, 128, 128, (16, 24, 24), False, "nhd"),
    (5, 7, 1, 64, 64, (32,), True, "nhd"), (33, 4, 4, 80, 40, (8, 6, 6), False, "hnd"),
    (130, 12, 12, 64, 32, (8, 8), True, None), (3, 3, 3, 6, 4, (1, 1), True, "nhd"), (257, 5, 1, 256, 256, (40, 44, 44), False, "hnd"),
    (19, 2, 2, 512, 512, (64,) * 4, True, "nhd"), (40, 64, 64, 128, 64, (0, 32), False, "nhd"),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,hq,hkv,dim,rot,sections,pairs,layout", ROPES)
def test_rope_append(cuda, dtype, tokens, hq, hkv, dim, rot, sections, pairs, layout):
    rng = np.random.default_rng(tokens * 7 + dim)
    torch.manual_seed(tokens + dim)
    T = TYPES[dtype]
    qkv = torch.randn(tokens, (hq + 2 * hkv) * dim, device="cuda", dtype=T)
    q, k, v = (x.view(tokens, -1, dim) for x in qkv.split([hq * dim, hkv * dim, hkv * dim], dim=1))
    length, axes = 50, len(sections)
    table = rng.standard_normal((length, rot)).astype(np.float32)
    pos = rng.integers(0, length, (axes, tokens))
    axis_of = serving.contiguous_axes(sections)
    assert len(axis_of) == rot // 2
    kw = {}
    if layout:
        block, blocks = 5, tokens // 5 + 3
        shape = (blocks, block, hkv, dim) if layout == "nhd" else (blocks, hkv, block, dim)
        kc, vc = (torch.full(shape, float("nan"), device="cuda", dtype=T) for _ in range(2))
        kw["k_cache"], kw["v_cache"] = (x if layout == "nhd" else x.transpose(1, 2) for x in (kc, vc))
        slots = rng.permutation(blocks * block)[:tokens]
        slots[tokens // 2] = -1 if tokens > 1 else slots[0]
        kw |= dict(slots=i32(slots), v=v)
    else:
        kw["v"] = None
    q_out, k_out = serving.rope_append(q, k, table=torch.from_numpy(table).cuda(), positions=i32(pos), axis_of=axis_of,
                                       interleaved=pairs, **kw)
    serving.synchronize()

    def close(got, x):  # two products and a sum in float32, then one rounding
        want, big = rope_ref(np64(x), table.astype(np.float64), pos, axis_of, pairs, rot)
        lim = 3 * 2.0**-24 * big * max(1.0, np.abs(table).max()) + U[dtype] * np.abs(want) * 1.01 + SMALLEST[dtype]
        assert (np.abs(np64(got) - want) <= lim).all()

    close(q_out, q)
    if not layout:
        close(k_out, k)
        return
    assert k_out is None
    flat_k, flat_v = (kw[n].reshape(-1, hkv, dim) for n in ("k_cache", "v_cache"))
    ok = slots >= 0
    at = torch.from_numpy(slots[ok]).cuda()
    keep = np.setdiff1d(np.arange(flat_k.shape[0]), slots[ok])
    assert torch.equal(flat_v[at], v[torch.from_numpy(ok).cuda()])
    assert torch.isnan(flat_k[torch.from_numpy(keep).cuda()]).all() and torch.isnan(flat_v[torch.from_numpy(keep).cuda()]).all()
    full = torch.empty_like(k)
    full.copy_(torch.zeros_like(k))
    written = torch.zeros_like(k)
    written[torch.from_numpy(ok).cuda()] = flat_k[at]
    want, big = rope_ref(np64(k), table.astype(np.float64), pos, axis_of, pairs, rot)
    lim = 3 * 2.0**-24 * big * max(1.0, np.abs(table).max()) + U[dtype] * np.abs(want) * 1.01 + SMALLEST[dtype]
    assert (np.abs(np64(written) - want)[ok] <= lim[ok]).all()


def test_rope_in_place_odd_strides_and_errors(cuda):
    table = torch.randn(9, 32, device="cuda")
    wide = torch.randn(6, 3, 37, device="cuda", dtype=torch.float16)  # heads 37 elements apart: no 16-byte rows
    q, k = wide[:, :2, 1:33], wide[:, 2:, 1:33]
    pos = i32(np.arange(6))
    a, b = serving.rope_append(q, k, None, table, pos)
    serving.rope_append(q, k, None, table, pos, q_out=q, k_out=k)
    serving.synchronize()
    assert torch.equal(q, a) and torch.equal(k, b)
    device_error(lambda: serving.rope_append(q, k, None, table, i32([0, 1, 2, 3, 4, 9])))
    cache = torch.zeros(2, 4, 1, 32, device="cuda", dtype=torch.float16)
    device_error(lambda: serving.rope_append(q, k, k, table, pos, slots=i32([0, 1, 2, 3, 4, 8]), k_cache=cache, v_cache=cache.clone()))
    with pytest.raises(ValueError):
        serving.rope_append(q, k, None, table.half(), pos)
    with pytest.raises(ValueError):
        serving.rope_append(q, k, None, table, pos, axis_of=(0,) * 15)
    with pytest.raises(ValueError):
        serving.rope_append(q, k, k, table, pos)
    with pytest.raises(_lib.NB2Error) as e:
        serving.rope_append(q[..., :16], k[..., :16], None, table, pos)  # rotates more than the head
    assert e.value.status == _lib.ERR_INVALID


# ---- tree attention -----------------------------------------------------------------------------------------------


class Batch:
    """A paged cache with its requests; every place that no token may read holds NaN."""

    def __init__(self, olds, news, hq, hkv, dim, block, dtype, layout="nhd", trees="random", seed=0, spread=1.5, empty=()):
        rng = np.random.default_rng(seed)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.old, self.new = np.asarray(olds), np.asarray(news)
        self.total = self.old + self.new
        self.off = np.concatenate([[0], np.cumsum(self.new)])
        self.hq, self.hkv, self.dim, self.block, self.dtype = hq, hkv, dim, block, dtype
        B, T = len(olds), int(self.off[-1])
        need = -(-self.total // block)
        blocks = int(need.sum()) + 3
        pool = rng.permutation(blocks)
        self.table = np.full((B, int(need.max()) + 1), -1)
        shape = (blocks, block, hkv, dim) if layout == "nhd" else (blocks, hkv, block, dim)
        kc, vc = (torch.full(shape, float("nan"), device="cuda", dtype=TYPES[dtype]) for _ in range(2))
        self.kc, self.vc = (x if layout == "nhd" else x.transpose(1, 2) for x in (kc, vc))
        at = 0
        self.k, self.v = [], []
        for r in range(B):
            self.table[r, :need[r]] = pool[at:at + need[r]]
            at += need[r]
            n = int(self.total[r])
            k, v = (torch.randn(n, hkv, dim, device="cuda", generator=gen).to(TYPES[dtype]) for _ in range(2))
            p = np.arange(n)
            b, o = torch.from_numpy(self.table[r, p // block]).cuda().long(), torch.from_numpy(p % block).cuda()
            self.kc[b, o], self.vc[b, o] = k, v
            self.k.append(np64(k))
            self.v.append(np64(v))
        self.q = (torch.randn(T, hq, dim, device="cuda", generator=gen) * spread).to(TYPES[dtype])
        self.words = max(1, -(-int(self.new.max()) // 32)) if trees else 0
        self.see = []
        bits = np.zeros((T, max(1, self.words) * 32), bool)
        for r in range(B):
            n = int(self.new[r])
            m = np.eye(n, dtype=bool)
            if trees is None:
                m = np.tril(np.ones((n, n), bool))
            else:
                for i, j in enumerate(tree_parents(rng, n, trees)):
                    if j >= 0:
                        m[i] |= m[j]
            for t in empty:
                if self.off[r] <= t < self.off[r + 1]:
                    m[t - self.off[r]] = False
            if trees:
                bits[self.off[r]:self.off[r + 1], :n] = m
            self.see.append(m)
        self.mask = i32(np.packbits(bits, axis=1, bitorder="little").view(np.int32)) if trees else None
        self.scale = dim**-0.5

    def run(self, **kw):
        kw = dict(tree_mask=self.mask, max_new=int(self.new.max()), return_lse=True) | kw
        return serving.tree_attention(kw.pop("q", self.q), self.kc, self.vc, i32(self.table), i32(self.total), i32(self.off), **kw)

    def check(self, out, lse, q=None):
        """Scores: dim products and sums in float32 (float32 inputs: each product by three, its rest below 2^-22);
        weights: exp and the sum over n places in float32, rounded to the cache's type for the second product."""
        q = np64(self.q if q is None else q)
        out, lse = np64(out), np64(lse)
        g, u = self.hq // self.hkv, U[self.dtype]
        assert np.isfinite(out).all()
        for r in range(len(self.old)):
            n, tot = int(self.new[r]), int(self.total[r])
            see = np.concatenate([np.ones((n, tot - n), bool), self.see[r]], 1)
            for h in range(self.hq):
                k, v = self.k[r][:, h // g], self.v[r][:, h // g]
                rows = slice(self.off[r], self.off[r + 1])
                s = q[rows, h] @ k.T * self.scale
                mag = np.abs(q[rows, h]) @ np.abs(k).T * self.scale
                eps = ((self.dim + 16) * 2.0**-23 * np.where(see, mag, 0)).max(1, initial=0.0)
                s[~see] = -np.inf
                top = s.max(1, initial=-np.inf)
                some = top > -np.inf
                assert np.array_equal(lse[rows, h] == -np.inf, ~some)
                assert (out[rows, h][~some] == 0).all()
                p = np.exp(s[some] - top[some, None])
                z = p.sum(1)
                want = p @ v / z[:, None]
                most = np.abs(v).max() if tot else 0.0
                lim = ((2 * eps[some] + 4 * u + (tot + 64) * 2.0**-23) * most)[:, None] + 1.01 * u * np.abs(want) + SMALLEST[self.dtype]
                if self.dtype == "f32":
                    lim = lim + 2.0**-20 * most
                assert (np.abs(out[rows, h][some] - want) <= lim).all()
                wl = top[some] + np.log(z)
                assert (np.abs(lse[rows, h][some] - wl) <= eps[some] + (tot + 64) * 2.0**-23 + 2.0**-22 * np.abs(wl)).all()


ATTN = [
    # olds, news, q heads, kv heads, dim, block, layout, trees
    ([0], [1], 1, 1, 8, 1, "nhd", "random"), ([1], [1], 2, 1, 64, 16, "nhd", "random"),
    ([0, 5, 17, 300], [3, 0, 1, 8], 8, 2, 128, 16, "nhd", "random"), ([1000, 31], [1, 1], 32, 8, 128, 16, "nhd", "random"),
    ([129, 127, 128], [5, 7, 64], 4, 4, 64, 32, "hnd", "random"), ([700, 63], [33, 40], 5, 1, 80, 24, "nhd", "random"),
    ([2100], [64], 8, 1, 128, 64, "nhd", "chain"), ([50, 900], [130, 2], 6, 2, 128, 7, "nhd", "star"),
    ([333, 40], [17, 90], 3, 1, 256, 16, "hnd", "random"), ([70, 0, 260], [20, 33, 1], 4, 2, 96, 128, "nhd", None),
    ([0, 0], [0, 4], 2, 2, 32, 16, "nhd", "random"), ([640, 1300, 64], [64, 64, 1], 32, 8, 128, 16, "nhd", "random"),
    ([4097], [16], 40, 8, 128, 64, "nhd", "random"), ([10], [300], 2, 1, 64, 16, "nhd", None), ([5000, 3], [1, 1], 16, 1, 64, 8, "nhd", None),
    ([3], [520], 7, 1, 128, 16, "nhd", "random"),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("olds,news,hq,hkv,dim,block,layout,trees", ATTN)
def test_tree_attention(cuda, dtype, olds, news, hq, hkv, dim, block, layout, trees):
    b = Batch(olds, news, hq, hkv, dim, block, dtype, layout, trees, seed=dim + hq)
    out, lse = b.run()
    serving.synchronize()
    b.check(out, lse)
    again, lse2 = b.run()
    serving.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, lse2)  # no order shows in the result


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_tree_attention_rows_that_see_nothing(cuda, dtype):
    b = Batch([0, 0, 40], [40, 3, 5], 8, 2, 64, 16, dtype, trees="random", empty=(0, 39, 41))
    out, lse = b.run()
    serving.synchronize()
    b.check(out, lse)
    assert (lse == -math.inf).all(1).nonzero().flatten().tolist() == [0, 39, 41]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("news,g", [([9, 40], 1), ([70, 40], 4)])
def test_tree_attention_masked_places_that_are_not_finite(cuda, dtype, news, g):
    """A drafted token whose key and value are infinite or NaN reaches the tokens that see it and no others."""
    b = Batch([50, 300], news, 2 * g, 2, 128, 16, dtype, trees="star")  # each drafted token sees itself only
    for r, i, val in ((0, 2, float("inf")), (1, 7, float("nan")), (1, 30, -float("inf"))):
        p = int(b.old[r]) + i
        block = int(b.table[r, p // 16])
        b.vc[block, p % 16] = val
        if val != val:
            b.kc[block, p % 16] = val
    out, lse = b.run()
    serving.synchronize()
    hit = [int(b.off[0]) + 2, int(b.off[1]) + 7, int(b.off[1]) + 30]
    assert not torch.isfinite(out[hit]).any()
    assert torch.isnan(lse[hit[1]]).all() and torch.isfinite(lse[hit[0]]).all()
    rest = [t for t in range(out.shape[0]) if t not in hit]
    clean = Batch([50, 300], news, 2 * g, 2, 128, 16, dtype, trees="star")
    want, want_lse = clean.run()
    serving.synchronize()
    assert torch.equal(out[rest], want[rest]) and torch.equal(lse[rest], want_lse[rest])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tree_attention_large_scores(cuda, dtype):
    """Scores of several hundred: the running maximum moves, and weights underflow."""
    b = Batch([500, 130], [9, 40], 4, 1, 128, 16, dtype, spread=40.0)
    out, lse = b.run()
    serving.synchronize()
    b.check(out, lse)


def test_tree_attention_strides_padding_and_bound(cuda):
    """q and out inside wider rows, tokens past the last request, and the default bound of new tokens."""
    b = Batch([64, 7], [5, 6], 4, 2, 64, 16, "bf16")
    T = 11
    wide = torch.zeros(T + 4, 8, 128, device="cuda", dtype=torch.bfloat16)
    wide[:T, :4, :64] = b.q
    dst = torch.full((T + 4, 6, 72), 7.0, device="cuda", dtype=torch.bfloat16)
    mask = torch.cat([b.mask, torch.full((4, b.words), -1, device="cuda", dtype=torch.int32)])
    out, lse = b.run(q=wide[:, :4, :64], tree_mask=mask, out=dst[:, 1:5, 8:], max_new=None)
    serving.synchronize()
    b.check(out[:T], lse[:T])
    assert (out[T:] == 0).all() and (lse[T:] == -math.inf).all()
    assert (dst[:, 0] == 7).all() and (dst[:, 5] == 7).all() and (dst[:, :, :8] == 7).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("olds,news,hq,hkv,dim,block", [
    ([40000], [3], 4, 1, 64, 16), ([30000], [12], 4, 1, 128, 16), ([30000, 0], [33, 2], 8, 1, 128, 64), ([9000], [70], 6, 3, 96, 32),
    ([12000, 7, 5000], [130, 0, 1], 2, 1, 64, 16), ([700 + 37 * i for i in range(24)], [40 - i for i in range(24)], 32, 8, 128, 16),
    ([400 + 91 * i for i in range(40)], [1 + i % 3 for i in range(40)], 16, 4, 64, 16), ([8000], [5], 3, 1, 256, 16),
])
def test_tree_attention_pieces(cuda, dtype, olds, news, hq, hkv, dim, block):
    """A few items in many pieces each, and many items in a few: two calls agree in every bit."""
    b = Batch(olds, news, hq, hkv, dim, block, dtype, seed=3)
    out, lse = b.run()
    again, lse2 = b.run()
    serving.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    b.check(out, lse)


@pytest.mark.parametrize("news,hq,hkv", [([70, 3], 4, 2), ([90, 130], 4, 1)])
@pytest.mark.parametrize("block", [8, 32, 256])
@pytest.mark.parametrize("pads", [(8, 8), (64, 64), (64, 192), (0, 72), (128, 0)])
def test_tree_attention_heads_inside_wider_ones(cuda, news, hq, hkv, block, pads):
    """Keys and values of many rows whose heads lie in wider ones, each its own, at any multiple of 16 bytes."""
    b = Batch([200, 77], news, hq, hkv, 128, block, "bf16")
    for name, pad in zip(("kc", "vc"), pads):
        x = getattr(b, name)
        wide = torch.full((*x.shape[:3], 128 + pad), float("nan"), device="cuda", dtype=x.dtype)
        wide[..., :128] = x
        setattr(b, name, wide[..., :128])
    out, lse = b.run()
    serving.synchronize()
    b.check(out, lse)


def test_tree_attention_offsets_past_32_bits(cuda):
    """Blocks more than 2^31 elements apart."""
    b = Batch([100], [9], 4, 1, 64, 64, "bf16")
    far = torch.empty(3 * 2**30 + 2**20, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.as_strided(far, tuple(b.kc.shape), (2**29 + 2**20 + 64 * i, 64, 64, 1), 0 if i else 2**19) for i in (0, 128))
    assert (b.kc.shape[0] - 1) * k.stride(0) > 2**31
    k.copy_(b.kc), v.copy_(b.vc)
    b.kc, b.vc = k, v
    out, lse = b.run()
    serving.synchronize()
    b.check(out, lse)


def test_tree_attention_on_another_stream_and_in_a_graph(cuda):
    b = Batch([200, 900, 3], [8, 16, 1], 8, 2, 128, 16, "bf16")
    args = [i32(b.table), i32(b.total), i32(b.off)]
    kw = dict(tree_mask=b.mask, max_new=16, return_lse=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        q = b.q * 1.0  # made on this stream, used on it with no wait in between
        out, lse = serving.tree_attention(q, b.kc, b.vc, *args, **kw)
        serving.synchronize()
    b.check(out, lse)
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out2, lse2 = serving.tree_attention(q, b.kc, b.vc, *args, **kw)
        for _ in range(2):
            out2.zero_()
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_tree_attention_wait_that_runs_out(cuda):
    """The many-row kernel's pipeline waits are bounded: past the bound it records a device error and ends, and the
    next call is as before."""
    b = Batch([700, 300], [40, 33], 8, 2, 128, 16, "bf16")
    out, lse = b.run()
    serving.synchronize()
    dev, L = serving.context(), _lib.lib()
    _lib.check(L.nb2_device_set_wait_bound(dev, 64))
    try:
        device_error(b.run)
    finally:
        _lib.check(L.nb2_device_set_wait_bound(dev, 0))
    again, lse2 = b.run()
    serving.synchronize()
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    b.check(again, lse2)


def test_tree_attention_negative_and_zero_scale(cuda):
    for scale in (-0.1, 0.0):
        for news in ([3, 1], [40, 33]):
            b = Batch([70, 300], news, 8, 2, 128, 16, "bf16")
            b.scale = scale
            out, lse = b.run(scale=scale)
            serving.synchronize()
            b.check(out, lse)


def test_tree_attention_no_requests(cuda):
    k = torch.zeros(2, 16, 2, 64, device="cuda")
    none = torch.zeros(0, device="cuda", dtype=torch.int32)
    out, lse = serving.tree_attention(torch.randn(3, 4, 64, device="cuda"), k, k, none.view(0, 1), none, i32([0]), return_lse=True)
    serving.synchronize()
    assert (out == 0).all() and (lse == -math.inf).all()
    p = serving.page_plan(none, none, none.view(0, 3), i32([4]), 16, 2)
    serving.synchronize()
    assert p.token_offsets.tolist() == [0] and p.slots.tolist() == [-1, -1] and p.free_head.tolist() == [0]


def test_tree_attention_errors(cuda):
    b = Batch([20, 30], [2, 3], 4, 2, 64, 16, "bf16")
    q, table, total, off = b.q, i32(b.table), i32(b.total), i32(b.off)
    kw = dict(tree_mask=b.mask, max_new=3)
    bad = table.clone()
    bad[1, 0] = b.kc.shape[0]
    device_error(lambda: serving.tree_attention(q, b.kc, b.vc, bad, total, off, **kw))
    bad[1, 0] = -1
    device_error(lambda: serving.tree_attention(q, b.kc, b.vc, bad, total, off, **kw))
    device_error(lambda: serving.tree_attention(q, b.kc, b.vc, table, i32([22, 2]), off, **kw))  # fewer places than new tokens
    device_error(lambda: serving.tree_attention(q, b.kc, b.vc, table, i32([22, 999]), off, **kw))  # more than the table holds
    device_error(lambda: serving.tree_attention(q, b.kc, b.vc, table, total, off, tree_mask=b.mask, max_new=2))
    out = serving.tree_attention(q, b.kc, b.vc, table, total, off, **kw)  # a good call after them
    serving.synchronize()
    b.check(out, b.run()[1])
    for wrong in (dict(q=q.half()), dict(q=q[:, :3].contiguous()), dict(q=q.double())):
        with pytest.raises((ValueError, _lib.NB2Error)):
            serving.tree_attention(wrong["q"], b.kc, b.vc, table, total, off, **kw)
    with pytest.raises(ValueError):
        serving.tree_attention(q, b.kc, b.vc, table.long(), total, off, **kw)
    with pytest.raises(ValueError):
        serving.tree_attention(q, b.kc, b.vc, table, total, off[:2], **kw)
    with pytest.raises(_lib.NB2Error) as e:
        serving.tree_attention(q[..., :60], b.kc[..., :60], b.vc[..., :60], table, total, off, **kw)
    assert e.value.status == _lib.ERR_INVALID


# ---- logit rules --------------------------------------------------------------------------------------------------


def logits_ref(x, row_request, prompt, output, rep, pres, freq, bias, masks, mask_rows):
    """(result, magnitude of what was added up)"""
    x = x.copy()
    big = np.abs(x)
    for i, r in enumerate(row_request):
        count = np.bincount(output[r], minlength=x.shape[1]) if len(output[r]) else np.zeros(x.shape[1])
        seen = count > 0
        seen[prompt[r]] = True
        y = x[i]
        y[seen] = np.where(y[seen] > 0, y[seen] / rep[r], y[seen] * rep[r])
        less = freq[r] * count + pres[r] * (count > 0)
        add = np.zeros(x.shape[1])
        for v, b in zip(*bias[r]):
            add[v] = b
        big[i] = np.maximum(big[i], np.abs(y)) + np.abs(freq[r] * count) + np.abs(pres[r]) + np.abs(add)
        y += add - less
        if masks is not None and mask_rows[i] >= 0:
            y[~masks[mask_rows[i]]] = -np.inf
    return x, big


LOGITS = [
    # requests, rows a request, vocab, longest history, biases, grammar
    (1, 1, 1, 0, 0, False), (1, 1, 33, 5, 3, True), (3, 2, 1000, 50, 7, True), (2, 1, 32003, 3000, 20, True), (5, 3, 4096, 9, 0, False),
    (2, 1, 128000, 20000, 300, True), (1, 1, 50257, 0, 1, True), (17, 1, 8191, 700, 64, True), (4, 9, 12289, 100, 5, True),
    (1, 1, 300001, 5000, 40, True),
]


@pytest.mark.parametrize("din,dout", [("f32", "f32"), ("bf16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("req,per,vocab,history,n_bias,grammar", LOGITS)
def test_logits_process(cuda, din, dout, req, per, vocab, history, n_bias, grammar):
    rng = np.random.default_rng(vocab + req)
    rows = req * per
    x = torch.from_numpy(rng.normal(0, 3, (rows, vocab))).to(TYPES[din]).cuda()
    rr = np.repeat(rng.permutation(req), per)
    prompt = [rng.integers(0, vocab, rng.integers(0, history + 1)) for _ in range(req)]
    output = [np.minimum(rng.geometric(0.01, rng.integers(0, history + 1)), vocab) - 1 for _ in range(req)]
    rep, pres, freq = (rng.uniform(a, b, req).astype(np.float32) for a, b in ((0.8, 1.5), (-0.3, 0.8), (0, 0.4)))
    bias = [(rng.integers(0, vocab, n_bias), rng.normal(0, 5, n_bias).astype(np.float32)) for _ in range(req)]  # some ids twice
    cat = lambda xs: (i32(np.concatenate([np.asarray(a) for a in xs] + [np.zeros(0, int)])), i32(np.concatenate([[0], np.cumsum([len(a) for a in xs])])))  # noqa: E731
    kw = {}
    masks = mask_rows = None
    if grammar:
        masks = rng.random((rows + 1, vocab)) < 0.5
        masks[0] = False  # a rule that allows nothing
        mask_rows = rng.integers(-1, rows + 1, rows)
        mask_rows[0] = 0
        full = np.zeros((rows + 1, -(-vocab // 32) * 32), bool)
        full[:, :vocab] = masks
        kw["grammar"] = (i32(np.packbits(full, axis=1, bitorder="little").view(np.int32)), i32(mask_rows))
        x[0, 0] = float("nan")
        x[0, vocab - 1] = float("inf")
    if n_bias:
        ids, off = cat([b[0] for b in bias])
        kw["bias"] = (ids, torch.from_numpy(np.concatenate([b[1] for b in bias])).cuda(), off)
    dev = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    got = serving.logits_process(x, prompt=cat(prompt), output=cat(output), row_request=i32(rr), repetition=dev(rep),
                                 presence=dev(pres), frequency=dev(freq), out_dtype=TYPES[dout], **kw)
    if din == dout:
        y = x.clone()
        assert serving.logits_process(y, prompt=cat(prompt), output=cat(output), row_request=i32(rr), repetition=dev(rep),
                                      presence=dev(pres), frequency=dev(freq), out=y, **kw) is y
        serving.synchronize()
        assert torch.equal(y.nan_to_num(), got.nan_to_num())
    serving.synchronize()
    with np.errstate(invalid="ignore"):
        want, big = logits_ref(np64(x), rr, prompt, output, rep.astype(float), pres.astype(float), freq.astype(float), bias, masks, mask_rows)
    got = np64(got)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine])
    # at most five float32 operations, then one rounding
    lim = 6 * 2.0**-24 * big[fine] + 1.01 * U[dout] * np.abs(want[fine]) + SMALLEST[dout]
    assert (np.abs(got[fine] - want[fine]) <= lim).all()


def test_logits_process_parts_and_errors(cuda):
    x = torch.randn(3, 500, device="cuda")
    assert torch.equal(serving.logits_process(x), x)
    sub = torch.randn(3, 700, device="cuda")[:, 3:503]  # rows that are not 16-byte aligned
    assert torch.equal(serving.logits_process(sub), sub)
    none = torch.randn(0, 500, device="cuda")
    assert serving.logits_process(none).shape == (0, 500)
    only = serving.logits_process(x, output=(i32([7, 7, 9]), i32([0, 2, 2, 3])), frequency=torch.full((3,), 0.5, device="cuda"))
    want = x.clone()
    want[0, 7] -= 1.0
    want[2, 9] -= 0.5
    assert torch.equal(only, want)
    off = i32([0, 1, 1, 1])
    device_error(lambda: serving.logits_process(x, prompt=(i32([500]), off)))
    device_error(lambda: serving.logits_process(x, output=(i32([-1]), off)))
    device_error(lambda: serving.logits_process(x, prompt=(i32([5]), i32([0, 2, 1, 1]))))
    device_error(lambda: serving.logits_process(x, prompt=(i32([5]), off), row_request=i32([0, 3, 1])))
    device_error(lambda: serving.logits_process(x, grammar=(torch.zeros(2, 16, device="cuda", dtype=torch.int32), i32([0, 1, 2]))))
    with pytest.raises(ValueError):
        serving.logits_process(x, grammar=(torch.zeros(3, 15, device="cuda", dtype=torch.int32), None))
    with pytest.raises(ValueError):
        serving.logits_process(x, prompt=(i32([5]), i32([0, 1])), requests=3)
    with pytest.raises(_lib.NB2Error) as e:
        serving.logits_process(x[:, :4].contiguous(), out=torch.empty(3, 4, device="cuda").as_strided((3, 4), (1, 1)))
    assert e.value.status == _lib.ERR_INVALID
