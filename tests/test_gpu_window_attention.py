"""Window attention with sinks against its definition in 64 bits (tolerances: long_context.exact_attention)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu


def run(gpu, b, window, sinks, **kw):
    d = b.to(gpu)
    return ops.window_attention(d.q, d.k_cache, d.v_cache, *b.meta(gpu), b.bs, b.scale, window, sinks, **kw)


def forms(b):
    """The ways to call with one batch."""
    yield "unknown packing", {}
    yield "packing on the host", dict(cu_seqlens=b.cu)
    yield "unsplit", dict(split=False)
    if (np.diff(b.cu) <= 1).all():
        yield "decode", dict(max_query_len=1)
        yield "decode, unsplit", dict(max_query_len=1, split=False)


def verify(gpu, b, window, sinks, what):
    exact, tol = LC.exact_attention(b, window, sinks)
    for name, kw in forms(b):
        print(f"[case] {what}: {name}", flush=True)
        LC.check(run(gpu, b, window, sinks, **kw), exact, tol, f"{what}, {name}")


# ctx, new, q_heads, kv_heads, head_dim, block size, window, sinks
CASES = [
    ([1], [1], 4, 2, 64, 16, 8, 4),                             # one key
    ([300], [1], 14, 2, 64, 256, 100, 4),                       # one token, both parts
    ([1500], [1], 28, 4, 128, 256, 1000, 70),                   # sinks over two chunks
    ([3000, 7, 65, 1, 640], [1] * 5, 28, 4, 128, 64, 512, 4),   # a ragged decode batch
    ([900, 128, 129], [1] * 3, 32, 8, 128, 16, 64, 1),          # window of whole chunks, small blocks
    ([700], [1], 16, 1, 128, 32, 100, 0),                       # no sinks, 16 heads a kv head
    ([700, 90], [1, 1], 40, 2, 128, 32, 100, 3),                # 20 heads a kv head
    ([257, 64, 33], [257, 64, 33], 28, 4, 128, 64, 50, 4),      # packed prompts
    ([500], [500], 8, 8, 64, 16, 130, 5),                       # one head a kv head
    ([333, 200], [120, 200], 14, 2, 64, 32, 64, 20),            # a chunk after cached keys
    ([600, 31, 400], [40, 1, 3], 32, 8, 128, 256, 200, 100),    # decode tokens packed with chunks
    ([90, 70], [90, 70], 6, 3, 80, 8, 33, 2),                   # other head and block sizes
    ([50, 40], [50, 2], 5, 1, 256, 24, 20, 3),
    ([45, 30], [45, 1], 3, 3, 37, 5, 11, 1),                    # odd everything
    ([200], [200], 4, 2, 128, 64, 1, 0),                        # each token sees itself
    ([200], [200], 4, 2, 128, 64, 0, 3),                        # sinks alone
    ([100], [100], 4, 2, 64, 16, 1 << 40, 0),                   # no window
    ([100], [100], 4, 2, 64, 16, 10, 1 << 40),                  # all keys are sinks
    ([130] * 20, [1] * 20, 28, 4, 128, 64, 100, 4),             # many sequences in a tile
    ([20, 140, 3, 64, 9], [20, 100, 2, 64, 9], 28, 4, 128, 16, 40, 2),
    ([1500, 900], [40, 21], 28, 4, 128, 64, 1200, 70),          # few tokens over a long window: key ranges
    ([1300], [33], 14, 2, 64, 16, 1 << 20, 0),
    ([70] * 50 + [100, 90] + [20] * 30, [1] * 50 + [100, 60] + [1] * 30, 28, 4, 128, 32, 48, 4),  # over 64 sequences
    ([40] * 66 + [150], [1, 2, 3] * 22 + [150], 8, 8, 64, 16, 30, 2),
    ([30] * 65, [30] * 65, 14, 2, 64, 16, 20, 1),
    ([300, 0, 65], [1, 0, 65], 28, 4, 128, 64, 64, 4),          # a sequence without tokens
]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ci", range(len(CASES)))
def test_window_attention(gpu, dt, ci):
    ctx, new, qh, kvh, hd, bs, window, sinks = CASES[ci]
    b = LC.make_batch(40 + ci, ctx, new, qh, kvh, hd, bs, dt, window, sinks)
    verify(gpu, b, window, sinks, f"case {ci}")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_no_window_is_paged_attention(gpu, dt):
    """With nothing masked the result is paged_attention's, within both tolerances."""
    b = LC.make_batch(3, [400, 70], [400, 1], 28, 4, 128, 64, dt)
    exact, tol = LC.exact_attention(b)
    d = b.to(gpu)
    want = ops.paged_attention(d.q, torch.nan_to_num(d.k_cache), torch.nan_to_num(d.v_cache), *b.meta(gpu), b.bs, b.scale)
    got = run(gpu, b, 1 << 20, 0)
    assert (np.abs((got.double() - want.double()).cpu().numpy()) <= 2 * tol).all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_rows_without_keys_are_zeros(gpu, dt):
    """Padding tokens (no keys, whatever their sequence) and masks that leave nothing."""
    b = LC.make_batch(5, [80, 64, 40], [1, 1, 1], 28, 4, 128, 64, dt, 32, 4)
    b.key_len[[0, 2]] = [0, -3]
    b.seq[2] = -1
    exact, tol = LC.exact_attention(b, 32, 4)
    for name, kw in forms(b):
        got = run(gpu, b, 32, 4, **kw)
        assert not got[0].any() and not got[2].any()
        LC.check(got, exact, tol, name)
    assert not run(gpu, b, 0, 0).any()
    e = b.to(gpu)
    assert ops.window_attention(e.q[:0], e.k_cache, e.v_cache, *[x[:0] for x in b.meta(gpu)[:2]], b.meta(gpu)[2], b.bs,
                                b.scale, 5).shape == (0, 28, 128)


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new", [150, 1], ids=["prompt", "decode"])
def test_masked_values_do_not_matter(gpu, dt, value, new):
    """Non-finite keys and values that some tokens of a tile see and others do not: only the first are
    touched, in the dimensions that hold them."""
    window, sinks = 40, 3
    b = LC.make_batch(9, [150, 60], [new, 1], 14, 2, 64, 16, dt, window, sinks)
    exact, tol = LC.exact_attention(b, window, sinks)
    for key in (100, 120):
        row = int(b.table[0, key // 16]) * 16 + key % 16
        b.v_cache[row, :, 5] = value
    sees = np.array([[s == 0 and LC.seen_keys(int(n), window, sinks)[key:key + 1].any() for key in (100, 120)]
                     for s, n in zip(b.seq, b.key_len)]).any(1)
    got = run(gpu, b, window, sinks, cu_seqlens=b.cu).double().cpu().numpy()
    touched = np.zeros(got.shape, bool)
    touched[sees, :, 5] = True
    assert not np.isfinite(got[touched]).any()
    assert (np.abs(got - exact) <= tol)[~touched].all()
    # keys: the tokens that do not see them
    b = LC.make_batch(9, [150, 60], [new, 1], 14, 2, 64, 16, dt, window, sinks)
    row = int(b.table[0, 120 // 16]) * 16 + 120 % 16
    b.k_cache[row] = value
    sees = np.array([s == 0 and n > 120 and n - window <= 120 for s, n in zip(b.seq, b.key_len)])
    got = run(gpu, b, window, sinks, cu_seqlens=b.cu).double().cpu().numpy()
    assert (np.abs(got - exact) <= tol)[~sees].all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("bs", [16, 64, 24])
@pytest.mark.parametrize("new", [70, 1], ids=["prompt", "decode"])
def test_bad_pages_give_nan_rows(gpu, dt, bs, new):
    """A seen key without a cache block: NaN; tokens that do not see it are right."""
    window, sinks = 30, 2
    b = LC.make_batch(11, [150, 33], [new, 1], 28, 4, 128, bs, dt, window, sinks)
    exact, tol = LC.exact_attention(b, window, sinks)
    blocks = b.k_cache.shape[0] // bs
    page = (150 - 40) // bs if new > 1 else 149 // bs
    sees = np.array([s == 0 and LC.seen_keys(int(n), window, sinks)[page * bs:(page + 1) * bs].any()
                     for s, n in zip(b.seq, b.key_len)])
    assert sees.any() and not sees.all()
    for bad in (-1, blocks, 2 ** 31 - 1):
        b.table[0, page] = bad
        for name, kw in forms(b):
            print(f"[case] bad page {bad}, {name}", flush=True)
            got = run(gpu, b, window, sinks, **kw).double().cpu().numpy()
            assert np.isnan(got[sees]).all()
            assert (np.abs(got - exact) <= tol)[~sees].all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("scale", [0.0, -0.1])
def test_scales_that_are_not_positive(gpu, dt, scale):
    b = LC.make_batch(14, [150, 33], [40, 1], 14, 2, 64, 16, dt, 30, 2)
    b.scale = scale
    q, b.scale = b.q, abs(scale)
    b.q = -q if scale < 0 else q * 0
    exact, tol = LC.exact_attention(b, 30, 2)  # of the positive scale and the negated queries
    b.q, b.scale = q, scale
    LC.check(run(gpu, b, 30, 2), exact, tol, f"scale {scale}")


def test_metadata_outside_the_tables(gpu):
    """A sequence that is no row of the tables, or more keys than a row holds: NaN rows, no read."""
    b = LC.make_batch(12, [150, 33], [1, 1], 28, 4, 128, 64, torch.float16, 30, 2)
    for seq, n in ((2, 20), (-1, 20), (0, 5000), (2 ** 31 - 1, 2 ** 31 - 1)):
        b.seq[0], b.key_len[0] = seq, n
        print(f"[case] sequence {seq}, {n} keys", flush=True)
        got = run(gpu, b, 30, 2, max_query_len=1)
        assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_strides_outputs_and_streams(gpu, dt):
    """q as columns of a packed row, an offset that breaks 16-byte alignment, a given out whose
    neighbours keep their values, and another stream than the default."""
    b = LC.make_batch(13, [200, 90], [200, 1], 8, 2, 64, 32, dt, 60, 4)
    exact, tol = LC.exact_attention(b, 60, 4)
    d, meta = b.to(gpu), b.meta(gpu)
    tokens = len(b.seq)
    for width, at in ((8 * 64 + 96, 32), (8 * 64 + 3, 1)):
        rows = torch.randn(tokens, width, device=gpu).to(dt)
        rows[:, at:at + 512] = d.q.view(tokens, 512)
        space = torch.full((tokens + 2, 8, 64), 7.0, dtype=dt, device=gpu)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            ops.window_attention(rows[:, at:at + 512].unflatten(1, (8, 64)), d.k_cache, d.v_cache, *meta, b.bs, b.scale,
                                 60, 4, out=space[1:-1])
        torch.cuda.current_stream().wait_stream(s)
        LC.check(space[1:-1], exact, tol, "strided")
        assert (space[0] == 7).all() and (space[-1] == 7).all()
    # caches that start off 16 bytes
    raw = torch.zeros(d.k_cache.numel() + 1, dtype=dt, device=gpu)
    k = raw[1:].view(d.k_cache.shape).copy_(d.k_cache)
    LC.check(ops.window_attention(d.q, k, d.v_cache, *meta, b.bs, b.scale, 60, 4), exact, tol, "unaligned cache")


def test_captured_calls(gpu):
    """Decode calls of two shapes captured one after the other: each replay equals the eager call,
    with eager work between, when the metadata changes."""
    bs = [LC.make_batch(20 + i, [900, 300], [1, 1], 28, 4, 128, 64, torch.bfloat16, 300 + i, 4) for i in range(2)]
    calls = []
    for i, b in enumerate(bs):
        d, meta = b.to(gpu), b.meta(gpu)
        run_it = lambda d=d, meta=meta, b=b, i=i: ops.window_attention(  # noqa: E731
            d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 300 + i, 4, max_query_len=1)
        eager = run_it()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run_it()
        calls.append((run_it, eager, g, out, d, meta))
    for _ in range(3):
        for run_it, eager, g, out, d, meta in calls:
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and torch.equal(run_it(), eager)
    for run_it, eager, g, out, d, meta in calls:
        meta[1][1] = 0  # the second sequence ends: its row becomes padding
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run_it()) and not out[1].any()


def test_large_offsets(gpu):
    """Cache rows past 2^32 bytes."""
    hd, kvh, bs = 128, 8, 64
    rows = (5 * 2 ** 30) // (hd * kvh * 2) // bs * bs  # 5 GiB of bf16 rows
    if torch.cuda.mem_get_info()[0] < 12 * 2 ** 30:
        pytest.skip("needs 12 GiB")
    b = LC.make_batch(30, [400], [130], 32, kvh, hd, bs, torch.bfloat16, 100, 4)
    exact, tol = LC.exact_attention(b, 100, 4)
    far = np.where(b.table >= 0, rows // bs - 20 + b.table % 20, -1)
    used = [(int(o), int(f)) for o, f in zip(b.table[0], far[0]) if 0 <= o < 100]
    assert len({f for _, f in used}) == len(used)
    k = torch.zeros((rows, kvh, hd), dtype=torch.bfloat16, device=gpu)
    v = torch.zeros((rows, kvh, hd), dtype=torch.bfloat16, device=gpu)
    for o, f in used:
        k[f * bs:(f + 1) * bs] = b.k_cache[o * bs:(o + 1) * bs].to(gpu)
        v[f * bs:(f + 1) * bs] = b.v_cache[o * bs:(o + 1) * bs].to(gpu)
    b.table = far
    meta = b.meta(gpu)
    for kw in ({}, dict(cu_seqlens=b.cu)):
        LC.check(ops.window_attention(b.q.to(gpu), k, v, *meta, bs, b.scale, 100, 4, **kw), exact, tol, "far rows")
    last = ops.window_attention(b.q[-1:].to(gpu), k, v, meta[0][-1:], meta[1][-1:], meta[2], bs, b.scale, 100, 4,
                                max_query_len=1)
    LC.check(last, exact[-1:], tol[-1:], "far rows, decode")
