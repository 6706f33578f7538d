"""Forks whose parents are not whole, and forks when pages run out."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC
from tests.test_gpu_cache_pages import Pool, host, make_caches, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("bad", [-1, -9, 8, 2 ** 31 - 1])
def test_a_parent_without_its_partial_page(gpu, dt, bad):
    """The parent's table holds no page of the cache where its partial page should be: nothing can be copied, so
    its child takes no page either (a page taken would show its last owner's keys), and another
    fork of the call gets the lowest free one."""
    table = np.array([[0, bad, -1], [1, 2, -1], [-1] * 3, [-1] * 3], np.int32)
    d = [torch.from_numpy(x).to(gpu) for x in (table, np.array([6, 7, 0, 0], np.int32),
                                               np.array([1, 1, 1, 0, 0, 0, 0, 0], np.int32))]
    caches = make_caches(gpu, 2, 8, (2, 64), 4, dt)
    want = host(caches, 8)
    new = ops.fork_pages(caches, *d, [0, 1], [2, 3], 4)
    assert new.tolist() == [-1, 3]
    assert d[0].tolist()[2:] == [[0, -1, -1], [1, 3, -1]] and d[1].tolist() == [6, 7, 6, 7]
    assert d[2].tolist() == [2, 2, 1, 1, 0, 0, 0, 0]
    for w in want:  # three rows of 128 values
        w[3, :3 * 128] = w[2, :3 * 128]
    same(caches, want, 8)
    # the child's missing key gives a NaN row, as its parent's does
    k, v = (c.view(-1, 2, 64).float() for c in caches)
    q = torch.randn(2, 4, 64, device=gpu)
    seq = torch.tensor([0, 2], dtype=torch.int32, device=gpu)
    n = torch.tensor([6, 6], dtype=torch.int32, device=gpu)
    assert torch.isnan(ops.window_attention(q, k, v, seq, n, d[0], 4, 0.1, 100)).all()


def test_the_last_pages_go_to_the_first_forks(gpu):
    """Two free pages for four forks, one of which needs none: the list by its restatement, entry by entry."""
    pool = Pool(4, 12, 4, 7, 16, {0: 40, 1: 32})
    caches = make_caches(gpu, 2, 7, (2, 64), 16, torch.float16)
    want, t = host(caches, 7), pool.gpu(gpu)
    free = np.flatnonzero(pool.ref == 0)
    assert len(free) == 2
    new = ops.fork_pages(caches, *t, [0, 1, 0, 0], [2, 3, 4, 5], 16).tolist()
    assert new == [int(free[0]), -1, int(free[1]), -2]
    assert new == pool.fork([0, 1, 0, 0], [2, 3, 4, 5], want)
    pool.check(t)
    same(caches, want, 7)
