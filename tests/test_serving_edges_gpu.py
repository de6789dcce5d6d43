"""The serving rows on the GPU where calls meet an edge: items of a single tile,
requests out of their bounds beside good ones, batches next to a launch limit,
replayed graphs, other GPUs and threads, views with odd strides. The plain
implementations and tolerances are those of test_serving_gpu."""

import math
import os
import subprocess
import sys
import threading
import time

import numpy as np
import pytest
import torch

from conftest import ROOT
from nert_b200 import _lib, serving
from test_serving_gpu import Batch, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("news", [(33, 40), (33, 64)])
def test_tree_attention_many_items_of_one_tile(cuda, dim, news):
    """Items of one tile of places one after another in a CTA: half of the many-row kernel has nothing to do in them."""
    rng = np.random.default_rng(5)
    new = rng.integers(news[0], news[1] + 1, 300)
    b = Batch(rng.integers(0, 64, 300), new, 4, 2, dim, 16, "bf16", seed=dim)
    out, lse = b.run()
    for _ in range(5):
        again, lse2 = b.run()
    serving.synchronize()
    assert np.array_equal(out.float().cpu().numpy(), again.float().cpu().numpy())
    assert np.array_equal(lse.cpu().numpy(), lse2.cpu().numpy())
    b.check(out, lse)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [72, 128])
def test_tree_attention_alternate_tiles(cuda, dtype, dim):
    """Up to 128 rows over one to a hundred tiles: the groups take alternate tiles from a ring of three."""
    b = Batch([5000, 0, 390, 1020, 12000, 100, 640], [100, 66, 128, 97, 70, 28, 65], 3, 3, dim, 32, dtype, seed=dim)
    out, lse = b.run()
    for _ in range(10):
        again, lse2 = b.run()
        assert (out == again).all() and (lse == lse2).all()
    serving.synchronize()
    b.check(out, lse)


PLAN_ALONE = """
import sys
import numpy as np, torch
from nert_b200 import _lib, serving
n = int(sys.argv[1])
i32 = lambda x: torch.tensor(np.asarray(x, np.int32), device="cuda")
new = np.arange(n) % 3
p = serving.page_plan(i32(np.full(n, 5)), i32(new), i32(np.arange(n)[:, None]), i32([0]), 16, int(new.sum()))
serving.synchronize()
r = np.repeat(np.arange(n), new)
i = np.concatenate([np.arange(x) for x in new])
assert np.array_equal(p.slots.cpu().numpy(), 16 * r + 5 + i)
assert np.array_equal(p.token_offsets.cpu().numpy(), np.concatenate([[0], np.cumsum(new)]))
"""


@pytest.mark.parametrize("batch", [6119, 6130, 6143, 6144, 8192])
def test_page_plan_of_any_batch_as_the_first_call(cuda, batch):
    """Around 48 KB of shared memory, static and dynamic part together: in a process of its own, where no larger
    call has raised the kernel's limit before."""
    done = subprocess.run([sys.executable, "-c", PLAN_ALONE, str(batch)], cwd=ROOT, capture_output=True, text=True,
                          env=os.environ | {"PYTHONPATH": ROOT}, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("dtype,dim,news,hq,hkv", [
    ("f32", 128, [200, 64, 40], 4, 1),  # joined by the mma.sync kernel's second launch, blocks of 64 rows
    ("bf16", 128, [200, 64, 64], 8, 1),  # by the tcgen05 kernel's, blocks of 256 rows
    ("f16", 64, [400, 90, 1], 1, 1),  # blocks of 128 rows
])
@pytest.mark.parametrize("first", [True, False])
def test_tree_attention_request_past_its_bound_beside_good_ones(cuda, dtype, dim, news, hq, hkv, first):
    """Only the request with more new tokens than max_new is refused: it gets out 0 and a device error, and those
    after it, split over many CTAs, what they get without it."""
    olds, most = [0, 30000, 20000], news[1]
    if not first:
        olds, news = olds[1:] + olds[:1], news[1:] + news[:1]
    b = Batch(olds, news, hq, hkv, dim, 16, dtype, seed=4)
    out = torch.full_like(b.q, 7.0)
    _, lse = b.run(max_new=most, out=out)
    with pytest.raises(_lib.NB2Error) as e:
        serving.synchronize()
    assert e.value.status == _lib.ERR_DEVICE
    r = 0 if first else 2
    rows = slice(int(b.off[r]), int(b.off[r + 1]))
    assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
    whole, whole_lse = b.run()
    serving.synchronize()
    b.check(whole, whole_lse)
    # the bad request's rows of the unbounded call, the others' of the bounded one
    out[rows], lse[rows] = whole[rows], whole_lse[rows]
    b.check(out, lse)


def _in_graph(stream, call, n=1):
    """A graph of n calls captured on a stream that has a context, and its last outputs."""
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        serving.context()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            for _ in range(n):
                out = call()
    return g, out


@pytest.mark.parametrize("dtype,olds,news", [
    ("bf16", [900, 2000, 60], [1, 1, 1]), ("f32", [700, 4000], [9, 12]), ("bf16", [3000, 900, 5000], [40, 33, 64]),
])
def test_graphs_of_one_stream_replayed_at_once(cuda, dtype, olds, news):
    """Graphs captured on one stream, replayed on two others beside calls on the first: each has pieces and
    tickets of its own. Every batch has items that several CTAs share."""
    bs = [Batch(olds, news, 16, 4, 128, 16, dtype, seed=s) for s in range(3)]
    args = [(b.q, b.kc, b.vc, i32(b.table), i32(b.total), i32(b.off)) for b in bs]
    calls = [lambda a=a, b=b: serving.tree_attention(*a, tree_mask=b.mask, max_new=max(news), return_lse=True) for a, b in zip(args, bs)]
    want = [c() for c in calls]
    serving.synchronize()
    for (out, lse), b in zip(want, bs):
        b.check(out, lse)
    first, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs = [_in_graph(first, c, 20) for c in calls[:2]]
    torch.cuda.synchronize()
    for _ in range(10):
        for (g, _), s in zip(graphs, others):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(first):
            for _ in range(20):
                eager = calls[2]()
        torch.cuda.synchronize()
        for (out, lse), (o, l) in zip([graphs[0][1], graphs[1][1], eager], want):
            assert torch.equal(out, o) and torch.equal(lse, l)
            out.zero_(), lse.zero_()
    with torch.cuda.stream(first):
        serving.synchronize()


def test_graphs_of_a_split_contraction_replayed_at_once(cuda):
    """Any row of the library on a caller's stream: here the partial sums of a Gemm that splits its long side."""
    from nert_b200._lib import check, ctypes, lib

    rows, n, k = 64, 64, 16384
    ws = [torch.randn(n, k, device="cuda") for _ in range(2)]
    xs = [torch.randn(rows, k, device="cuda") for _ in range(2)]

    def gemm(x, packed, y):
        check(lib().nb2_gemm_run_packed(serving.context(), x.data_ptr(), packed.data_ptr(), None, 0, y.data_ptr(), rows, n, k, 0,
                                        1.0, 1.0, _lib.ACT_NONE))
        return y

    packs = []
    for w in ws:
        size = ctypes.c_int64()
        check(lib().nb2_gemm_packed_size(n, k, ctypes.byref(size)))
        packs.append(torch.empty(size.value, device="cuda", dtype=torch.uint8))
        check(lib().nb2_gemm_pack(serving.context(), w.data_ptr(), n, k, 1, packs[-1].data_ptr()))
    ys = [torch.empty(rows, n, device="cuda") for _ in range(2)]
    want = [gemm(x, p, torch.empty_like(ys[0])) for x, p in zip(xs, packs)]
    slices = ctypes.c_int()
    check(lib().nb2_device_last_contraction(serving.context(), None, None, ctypes.byref(slices), None, None))
    assert slices.value > 1
    serving.synchronize()
    first, others = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs = [_in_graph(first, lambda x=x, p=p, y=y: gemm(x, p, y), 20)[0] for x, p, y in zip(xs, packs, ys)]
    for _ in range(10):
        torch.cuda.synchronize()
        for g, s in zip(graphs, others):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for y, w in zip(ys, want))
    for y, x, w in zip(ys, xs, ws):
        ref = x.double() @ w.double().T
        assert ((y.double() - ref).abs().max() / ref.abs().max()).item() <= 1e-4


def test_graphs_give_their_workspace_back(cuda):
    """A workspace belongs to a graph as long as it lives: the next capture takes one that a dead graph had."""
    b = Batch([30000], [12], 4, 1, 128, 16, "bf16")
    args = (b.q, b.kc, b.vc, i32(b.table), i32(b.total), i32(b.off))
    want = serving.tree_attention(*args, tree_mask=b.mask, max_new=12)
    stream = torch.cuda.Stream()
    left = []
    for _ in range(40):
        g, out = _in_graph(stream, lambda: serving.tree_attention(*args, tree_mask=b.mask, max_new=12))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        del g, out
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        left.append(torch.cuda.mem_get_info()[0])
    assert left[5] - left[-1] < 32 << 20  # one workspace is 10 MB


def test_errors_of_a_graph_replayed_on_another_stream(cuda):
    """What a replayed graph records is raised where its stream is waited for, once, and not by the next replay."""
    old, new, table = i32([3, 4]), i32([1, 1]), i32([[0], [1]])
    free, stream = i32([2]), torch.cuda.Stream()
    g, plan = _in_graph(stream, lambda: serving.page_plan(old, new, table, free, 16, 2))
    g.replay()
    serving.synchronize()
    assert plan.slots.tolist() == [3, 20]
    old.fill_(-1)
    g.replay()
    with pytest.raises(_lib.NB2Error) as e:
        serving.synchronize()
    assert e.value.status == _lib.ERR_DEVICE
    serving.synchronize()
    old.copy_(i32([5, 6]))
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        g.replay()
        serving.synchronize()
    with torch.cuda.stream(stream):
        serving.synchronize()
    assert plan.slots.tolist() == [5, 22]
    # a call's own error is its stream's, as before
    with torch.cuda.stream(other):
        serving.page_plan(i32([-1]), i32([1]), i32([[0]]), free, 16, 1)
        torch.cuda.synchronize()
    serving.synchronize()
    with torch.cuda.stream(other), pytest.raises(_lib.NB2Error):
        serving.synchronize()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two GPUs: the current one and another")
def test_the_current_gpu_stays_the_callers(cuda):
    """Calls on another GPU's tensors leave torch's current GPU as it was, with the first use of a stream or later."""
    there = torch.device("cuda:1")
    ints = lambda x: torch.tensor(x, device=there, dtype=torch.int32)  # noqa: E731
    half = lambda *shape: torch.zeros(*shape, device=there, dtype=torch.float16)  # noqa: E731
    torch.cuda.set_device(0)
    for _ in range(2):
        for call in (
            lambda: serving.context(there),
            lambda: serving.page_plan(ints([0]), ints([1]), ints([[0]]), ints([0]), 16, 1),
            lambda: serving.rope_append(half(1, 1, 8), half(1, 1, 8), None, torch.zeros(4, 8, device=there), ints([0])),
            lambda: serving.tree_attention(half(1, 1, 64), half(1, 16, 1, 64), half(1, 16, 1, 64), ints([[0]]), ints([1]), ints([0, 1])),
            lambda: serving.logits_process(half(1, 8)),
            lambda: serving.synchronize(there),
        ):
            call()
            assert torch.cuda.current_device() == 0 and torch.zeros(1, device="cuda").device.index == 0


def test_other_threads_run_while_one_waits(cuda):
    """synchronize() waits without the interpreter's lock, in several threads too, and each error is raised once."""
    serving.synchronize()
    turns, stop = [0], threading.Event()

    def count():
        while not stop.wait(0.001):
            turns[0] += 1

    other = threading.Thread(target=count)
    other.start()
    try:
        torch.cuda._sleep(600_000_000)  # about 0.3 s
        before = turns[0]
        serving.synchronize()
        assert turns[0] - before > 20
    finally:
        stop.set()
        other.join()

    raised = []

    def wait():
        try:
            serving.synchronize()
        except _lib.NB2Error as e:
            raised.append(e.status)

    for _ in range(5):
        serving.page_plan(i32([-1]), i32([1]), i32([[0]]), i32([0]), 16, 1)
        threads = [threading.Thread(target=wait) for _ in range(4)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert raised == [_lib.ERR_DEVICE]
        raised.clear()


def _odd_ones(x, *dims):
    """x with a stride of 3 in those of its dimensions that have one element."""
    return x.as_strided(x.shape, [3 if d in dims and n == 1 else s for d, (s, n) in enumerate(zip(x.stride(), x.shape))])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("olds,news,hq,hkv,block", [
    ([20], [1], 1, 1, 1), ([70, 5], [2, 9], 4, 1, 16), ([3], [9], 8, 1, 16), ([300], [90], 1, 1, 16), ([10], [100], 2, 1, 256),
])
def test_any_stride_of_a_dimension_of_one(cuda, dtype, olds, news, hq, hkv, block):
    b = Batch(olds, news, hq, hkv, 64, block, dtype)
    want, want_lse = b.run()
    serving.synchronize()
    b.check(want, want_lse)
    if block == 256:  # one block holds the request
        b.kc, b.vc = (c[int(b.table[0, 0]):][:1] for c in (b.kc, b.vc))
        b.table[:] = 0
    b.q = _odd_ones(b.q, 0, 1)
    b.kc, b.vc = _odd_ones(b.kc, 0, 1, 2), _odd_ones(b.vc, 0, 1, 2)
    out, lse = b.run(out=_odd_ones(torch.empty_like(want), 0, 1))
    serving.synchronize()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)

    # and the rotary row's, in values equal to those of plain views
    n, pos, table = b.q.shape[0], i32(np.arange(b.q.shape[0])), torch.randn(b.q.shape[0], 64, device="cuda")
    k = torch.randn(n, 1, 64, device="cuda").to(b.q.dtype)
    q0, k0 = serving.rope_append(b.q.contiguous(), k, None, table, pos)
    q1, k1 = serving.rope_append(b.q, _odd_ones(k, 0, 1), None, table, pos)
    serving.synchronize()
    assert torch.equal(q0, q1) and torch.equal(k0, k1)


@pytest.mark.parametrize("dtype,olds,news", [("bf16", [3000, 10], [1, 1]), ("f32", [900, 40, 0], [9, 12, 3]), ("f16", [5000, 70], [64, 33])])
def test_tree_attention_over_its_queries(cuda, dtype, olds, news):
    b = Batch(olds, news, 8, 2, 128, 16, dtype)
    want, want_lse = b.run()
    out, lse = b.run(out=b.q)
    serving.synchronize()
    assert out.data_ptr() == b.q.data_ptr() and torch.equal(out, want) and torch.equal(lse, want_lse)


def test_logit_lists_and_masks_that_hold_nothing(cuda):
    """What points into an empty list or set of masks is checked as into any other."""
    x = torch.randn(2, 64, device="cuda")
    none, words = i32([]), torch.zeros(0, 2, device="cuda", dtype=torch.int32)
    values = torch.zeros(0, device="cuda")
    got = serving.logits_process(x, prompt=(none, i32([0, 0, 0])), output=(none, i32([0, 0, 0])),
                                 bias=(none, values, i32([0, 0, 0])), grammar=(words, i32([-1, -1])))
    serving.synchronize()
    assert torch.equal(got, x)
    for wrong in (dict(prompt=(none, i32([0, 1, 1]))), dict(output=(none, i32([0, 0, 3]))),
                  dict(bias=(none, values, i32([0, 2, 2]))), dict(grammar=(words, i32([-1, 0]))), dict(grammar=(words, None))):
        serving.logits_process(x, **wrong)
        with pytest.raises(_lib.NB2Error) as e:
            serving.synchronize()
        assert e.value.status == _lib.ERR_DEVICE


@pytest.mark.parametrize("val", [3.4028234663852886e38, -3.4028234663852886e38, 3.4015e38, 3.4e38])
def test_largest_values_in_places_that_are_not_seen(cuda, val):
    """Finite float32 values up to the largest in one drafted token's row reach the token that sees it and no others."""
    news = [9, 40]
    b, clean = (Batch([50, 300], news, 2, 2, 128, 16, "f32", trees="star") for _ in range(2))
    t, r, i = 9 + 7, 1, 7
    p = int(b.old[r]) + i
    b.vc[int(b.table[r, p // 16]), p % 16, :, ::5] = val
    b.kc[int(b.table[r, p // 16]), p % 16, 1, 3] = val
    out, lse = b.run()
    want, want_lse = clean.run()
    serving.synchronize()
    rest = [x for x in range(out.shape[0]) if x != t]
    assert torch.equal(out[rest], want[rest]) and torch.equal(lse[rest], want_lse[rest])
    # the token that sees it: its weight (head 0, whose key is as it was) times the value and the sum of the others
    q, k = b.q[t, 0].double().cpu().numpy(), b.k[r][:, 0]
    see = np.arange(int(b.total[r])) < int(b.old[r])
    see[p] = True
    s = np.where(see, k @ q * b.scale, -np.inf)
    w = np.exp(s - s.max())
    w /= w.sum()
    got = out[t, 0].double().cpu().numpy()
    wanted = w @ b.v[r][:, 0]
    wanted[::5] += w[p] * (val - b.v[r][p, 0, ::5])
    assert np.isfinite(got).all()
    # scores and sums as in Batch.check; its largest value is the planted one in those columns
    most = np.where(np.arange(128) % 5 == 0, abs(val) * w[p] + 10, 10)
    eps = 2 * (128 + 16) * 2.0**-23 * (np.abs(k) @ np.abs(q))[see].max() * b.scale + (int(b.total[r]) + 64) * 2.0**-23 + 2.0**-20
    assert (np.abs(got - wanted) <= (eps + 4 * 2.0**-24) * most).all()
