"""Prefix attention where a token of a group cannot stand for the others: padding, sequences that have ended,
sequences that are no row of the tables, tokens that end inside the prefix.  Every other token of the group
keeps its result, as with share=False."""
from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC
from tests.test_gpu_prefix_attention import run, shared_batch

pytestmark = pytest.mark.gpu


def agree(gpu, b, prefix, start, exact, tol, rows, what):
    """Rows `rows` of the call are right, with the prefix shared and without."""
    for kw in ({}, dict(share=False)):
        print(f"[case] {what} {kw}", flush=True)
        got = run(gpu, b, prefix, start, **kw)
        LC.check(got[rows], exact[rows], tol[rows], f"{what} {kw}")
        yield got


def batch(dt, sizes, prefix, tails, seed=200, heads=(28, 4, 128, 64)):
    tails = [tails[i % len(tails)] for i in range(sum(sizes))]
    b, start = shared_batch(seed, sizes, prefix, tails, *heads[:3], heads[3], dt)
    return b, start, *LC.exact_attention(b)


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("heads", [(28, 4, 128, 64), (14, 2, 64, 16), (40, 2, 64, 32)])
@pytest.mark.parametrize("how", ["padding", "ended", "freed row", "no row", "short"])
def test_first_token_of_a_group(gpu, dt, heads, how):
    """The first tokens of a group: padding rows, ended sequences, and tokens with few keys."""
    b, start, exact, tol = batch(dt, [30, 4], [300, 70], [1, 5, 90], heads=heads)
    out = []
    for t in (0, 1, 30):
        if how == "padding":        # no keys, whatever the sequence
            b.seq[t], b.key_len[t] = -1, 0
        elif how == "ended":        # its pages given back
            b.table[t], b.key_len[t] = -1, 0
        elif how == "freed row":    # the same, with the key count of the step before
            b.table[t] = -1
        elif how == "no row":
            b.seq[t] = 1000
        else:
            b.key_len[t] = 3
            b.table[t, 1:] = -1
        out.append(t)
    if how == "short":
        exact, tol = LC.exact_attention(b)
        out = []
    live = np.setdiff1d(np.arange(len(b.seq)), out)
    for got in agree(gpu, b, [300, 70], start, exact, tol, live, how):
        if how in ("padding", "ended"):
            assert not got[out].any()
        elif out:
            assert torch.isnan(got[out]).all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_a_token_without_a_row_ends_inside_the_prefix(gpu, dt):
    """Its keys are the prefix's alone: NaN all the same, wherever it stands; so too if no token has a row."""
    for at in (0, 4, 8):
        b, start, exact, tol = batch(dt, [9], [200], [3, 40])
        b.seq[at], b.key_len[at] = 77, 150
        live = np.setdiff1d(np.arange(9), at)
        for got in agree(gpu, b, [200], start, exact, tol, live, f"token {at}"):
            assert torch.isnan(got[at]).all()
    b.seq[:], b.key_len[:] = -1, 150
    b.key_len[3] = 0
    got = run(gpu, b, [200], start)
    assert torch.isnan(got[[0, 1, 2, 4, 5, 6, 7, 8]]).all() and not got[3].any()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_a_page_that_one_table_lacks(gpu, dt):
    """A page of the prefix gone from one sequence's table: that sequence's row, no other one."""
    for s in (0, 3):
        b, start, exact, tol = batch(dt, [7], [260], [2, 9, 30])
        b.table[s, 1] = -1
        live = np.setdiff1d(np.arange(7), s)
        got = run(gpu, b, [260], start, share=False)
        LC.check(got[live], exact[live], tol[live], f"sequence {s} alone")
        assert torch.isnan(got[s]).all()
        got = run(gpu, b, [260], start)
        LC.check(got[live], exact[live], tol[live], f"sequence {s}")


@pytest.mark.parametrize("dt", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_tiles_of_padding(gpu, dt):
    """A group whose first tile holds padding alone, and whose second begins with it."""
    b, start, exact, tol = batch(dt, [50], [500], [1, 20])
    b.seq[:21], b.key_len[:21] = -1, 0
    for got in agree(gpu, b, [500], start, exact, tol, np.arange(21, 50), "21 rows of padding"):
        assert not got[:21].any()


def test_captured_group_whose_first_sequence_ends(gpu):
    """A captured decode step over samples of one prompt; they end one after the other between replays."""
    b, start, exact, tol = batch(torch.bfloat16, [12], [400], [5, 60, 33, 1])
    d, meta = b.to(gpu), b.meta(gpu)
    call = lambda **kw: ops.prefix_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 400, **kw)  # noqa: E731
    call()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = call()
    table, key_len = meta[2], meta[1]
    ref = torch.ones(b.k_cache.shape[0] // b.bs, dtype=torch.int32, device=gpu) * 12
    lens = key_len.clone()
    for ended in (0, 1, 2):
        ops.free_pages(table, lens, ref, [ended], b.bs)
        key_len.copy_(lens)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        live = np.arange(ended + 1, 12)
        LC.check(out[live], exact[live], tol[live], f"{ended + 1} ended")
        assert not out[:ended + 1].any()
        assert torch.equal(out, call())
        LC.check(call(share=False)[live], exact[live], tol[live], "alone")
