"""The serving rows on the GPU where calls meet an edge: items of a single tile,
requests out of their bounds beside good ones, batches next to a launch limit,
replayed graphs, other GPUs and threads, views with odd strides. The plain
implementations and tolerances are those of test_serving_gpu."""

import numpy as np
import pytest

from nert_b200 import serving
from test_serving_gpu import Batch

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
