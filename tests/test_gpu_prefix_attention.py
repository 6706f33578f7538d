"""Prefix attention against its definition in 64 bits (tolerances: long_context.exact_attention)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu


def shared_batch(seed, sizes, prefix, tails, q_heads, kv_heads, hd, bs, dt, new=None) -> tuple[LC.Batch, np.ndarray]:
    """Groups of sequences with prefix[g] keys in common, as forks leave them: full pages shared, the page
    that the prefix ends in each sequence's own.  Returns (batch, group_start)."""
    group = np.repeat(np.arange(len(sizes)), sizes)
    ctx = np.array([prefix[g] + t for g, t in zip(group, tails)])
    new = np.ones(len(ctx), np.int64) if new is None else np.asarray(new)
    b = LC.make_batch(seed, ctx, new, q_heads, kv_heads, hd, bs, dt)
    first = np.concatenate([[0], np.cumsum(sizes)])
    for s, g in enumerate(group):
        lead, full = first[g], prefix[g] // bs
        b.table[s, :full] = b.table[lead, :full]
        if prefix[g] % bs and s != lead and prefix[g] <= min(ctx[s], ctx[lead]):
            a, c = int(b.table[lead, full]) * bs, int(b.table[s, full]) * bs
            b.k_cache[c:c + prefix[g] % bs] = b.k_cache[a:a + prefix[g] % bs]
            b.v_cache[c:c + prefix[g] % bs] = b.v_cache[a:a + prefix[g] % bs]
    start = np.concatenate([[0], np.cumsum([new[group == g].sum() for g in range(len(sizes))])])
    return b, start


def run(gpu, b, prefix, start, **kw):
    d = b.to(gpu)
    return ops.prefix_attention(d.q, d.k_cache, d.v_cache, *b.meta(gpu), b.bs, b.scale, prefix, start, **kw)


# sizes, prefixes, tails (cycled), q_heads, kv_heads, head_dim, block size
CASES = [
    ([1], [1], [1], 4, 2, 64, 16),
    ([8], [100], [1, 30, 64], 14, 2, 64, 16),
    ([5], [64], [3, 70], 28, 4, 128, 64),                     # the prefix ends with a page and a chunk
    ([40], [700], [1, 5, 130], 28, 4, 128, 256),              # several tiles
    ([3, 1, 20], [200, 33, 65], [1, 17, 90], 32, 8, 128, 16),
    ([2, 0, 4], [50, 40, 0], [6, 1], 8, 8, 64, 32),           # an empty group, one without a prefix
    ([6], [300], [2, 9], 16, 1, 128, 64),                     # 16 heads a kv head
    ([4], [130], [5, 1], 40, 2, 64, 32),                      # 20 heads a kv head
    ([3, 2], [60, 45], [4, 20], 6, 3, 80, 8),                 # other head and block sizes
    ([3], [37], [4, 9], 3, 3, 37, 5),
    ([4], [50], [6, 2], 5, 1, 256, 24),
    ([150], [129], [1, 2, 3], 4, 4, 64, 16),                  # one head a kv head: more than a tile of tokens
    ([2] * 70, [20, 33] * 35, [1, 8], 14, 2, 64, 16),         # more groups than one launch takes
]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ci", range(len(CASES)))
def test_prefix_attention(gpu, dt, ci):
    sizes, prefix, tails, qh, kvh, hd, bs = CASES[ci]
    tails = [tails[i % len(tails)] for i in range(sum(sizes))]
    b, start = shared_batch(60 + ci, sizes, prefix, tails, qh, kvh, hd, bs, dt)
    exact, tol = LC.exact_attention(b)
    for kw in ({}, dict(share=False)):
        print(f"[case] {ci} {kw}", flush=True)
        LC.check(run(gpu, b, prefix, start, **kw), exact, tol, f"case {ci} {kw}")


# most of the work in the tiles, in the tokens' own keys, and neither; groups of unlike lengths
LEVELS = [
    ([120], [1500], [1, 2], 28, 4, 128, 64),
    ([30, 2], [64, 900], [700, 3], 32, 8, 128, 32),
    ([5, 34, 7], [72, 1024, 1317], [2, 1], 32, 8, 128, 256),
    ([60], [1], [400, 1, 90], 14, 2, 64, 16),
    ([1, 33], [1999, 30], [1, 40], 14, 2, 64, 32),
]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ci", range(len(LEVELS)))
def test_work_of_both_kinds(gpu, dt, ci):
    sizes, prefix, tails, qh, kvh, hd, bs = LEVELS[ci]
    tails = [tails[i % len(tails)] for i in range(sum(sizes))]
    b, start = shared_batch(110 + ci, sizes, prefix, tails, qh, kvh, hd, bs, dt)
    exact, tol = LC.exact_attention(b)
    LC.check(run(gpu, b, prefix, start), exact, tol, f"levels {ci}")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_several_tokens_a_sequence(gpu, dt):
    """Chunks after the prefix, and tokens that end inside it, at its end and at no key."""
    b, start = shared_batch(80, [3, 2], [150, 64], [20, 9, 31, 12, 70], 28, 4, 128, 16, dt, new=[20, 1, 31, 5, 7])
    b.key_len[3], b.key_len[20], b.key_len[30], b.key_len[55] = 100, 150, 0, 64
    exact, tol = LC.exact_attention(b)
    got = run(gpu, b, [150, 64], start)
    LC.check(got, exact, tol, "tokens of several lengths")
    assert not got[30].any()


def test_one_prefix_for_all_tokens(gpu):
    b, _ = shared_batch(81, [7], [90], [1, 2, 3, 4, 5, 6, 7], 28, 4, 128, 64, torch.bfloat16)
    exact, tol = LC.exact_attention(b)
    LC.check(run(gpu, b, 90, None), exact, tol, "an int")
    for shorter in (0, 1, 63, 64, 89):  # a caller may name fewer keys than are shared
        LC.check(run(gpu, b, shorter, None), exact, tol, f"{shorter} of 90 keys")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_values_of_other_sequences_do_not_matter(gpu, dt):
    """A non-finite value in one sequence's own keys, and one behind the prefix in the leader's page."""
    b, start = shared_batch(82, [6], [100], [10, 20, 3, 40, 5, 6], 14, 2, 64, 16, dt)
    exact, tol = LC.exact_attention(b)
    b.v_cache[int(b.table[0, 6]) * 16 + 101 % 16] = float("nan")  # key 101 of the first sequence
    b.k_cache[int(b.table[3, 7]) * 16 + 120 % 16] = float("inf")
    got = run(gpu, b, [100], start).double().cpu().numpy()
    assert np.isnan(got[0]).all()
    for s in (1, 2, 4, 5):
        assert (np.abs(got[s] - exact[s]) <= tol[s]).all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("share", [True, False])
def test_bad_pages_give_nan_rows(gpu, dt, share):
    """A bad page among a sequence's own keys: its row alone; one in the prefix: the group's rows."""
    b, start = shared_batch(83, [3, 2], [64, 48], [30, 20, 10, 9, 40], 28, 4, 128, 16, dt)
    exact, tol = LC.exact_attention(b)
    blocks = b.k_cache.shape[0] // 16
    for bad in (-1, blocks, 2 ** 31 - 1):
        c = LC.dataclasses.replace(b, table=b.table.copy())
        c.table[1, 5] = bad
        c.table[3:, 1] = bad
        print(f"[case] bad page {bad} share={share}", flush=True)
        got = run(gpu, c, [64, 48], start, share=share).double().cpu().numpy()
        assert np.isnan(got[[1, 3, 4]]).all()
        assert (np.abs(got - exact) <= tol)[[0, 2]].all()
    c = LC.dataclasses.replace(b, seq=b.seq.copy())
    c.seq[1] = 99
    got = run(gpu, c, [64, 48], start, share=share).double().cpu().numpy()
    assert np.isnan(got[1]).all() and (np.abs(got - exact) <= tol)[[0, 2, 3, 4]].all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_strides_and_outputs(gpu, dt):
    b, _ = shared_batch(84, [9], [77], [4, 12, 3, 9, 1, 30, 2, 5, 8], 8, 2, 64, 16, dt)
    exact, tol = LC.exact_attention(b)
    d, meta = b.to(gpu), b.meta(gpu)
    for width, at in ((8 * 64 + 96, 32), (8 * 64 + 3, 1)):
        rows = torch.randn(9, width, device=gpu).to(dt)
        rows[:, at:at + 512] = d.q.view(9, 512)
        space = torch.full((11, 8, 64), 7.0, dtype=dt, device=gpu)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.prefix_attention(rows[:, at:at + 512].unflatten(1, (8, 64)), d.k_cache, d.v_cache, *meta, b.bs, b.scale,
                                 77, out=space[1:-1])
        torch.cuda.current_stream().wait_stream(s)
        LC.check(space[1:-1], exact, tol, "strided")
        assert (space[0] == 7).all() and (space[-1] == 7).all()


def test_captured_calls(gpu):
    """Two captured calls, replayed with eager work between; key counts change between replays."""
    calls = []
    for i in range(2):
        b, start = shared_batch(86 + i, [12], [400 + i], [5, 60, 33, 1] * 3, 28, 4, 128, 64, torch.float16)
        d, meta = b.to(gpu), b.meta(gpu)
        run_it = lambda d=d, meta=meta, b=b, i=i: ops.prefix_attention(  # noqa: E731
            d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 400 + i)
        eager = run_it()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run_it()
        calls.append((run_it, eager, g, out, meta))
    for _ in range(3):
        for run_it, eager, g, out, meta in calls:
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and torch.equal(run_it(), eager)
    for run_it, eager, g, out, meta in calls:
        meta[1][5] -= 3
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run_it()) and not torch.equal(out[5], eager[5])
