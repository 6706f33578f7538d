"""Paged attention over 4-bit caches against its definition in 64 bits (tolerances: kv4.exact_attention)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC

pytestmark = pytest.mark.gpu


def forms(b):
    """The ways to call with one batch: (name, arguments, whether P may be rounded to fp16)."""
    some = b.q.shape[0] * (b.q.shape[1] // b.k_cache.shape[1]) > 16 and b.q.dtype != torch.float32
    yield "unknown packing", {}, some
    yield "packing on the host", dict(cu_seqlens=b.cu), some
    yield "unsplit", dict(split=False), some
    if (np.diff(b.cu) <= 1).all():
        yield "decode", dict(max_query_len=1), False
        yield "decode, unsplit", dict(max_query_len=1, split=False), False


def verify(gpu, b, kc, vc, what):
    exact = {some: kv4.exact_attention(b, some) for some in {f[2] for f in forms(b)}}
    q, k, v = b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    for name, kw, some in forms(b):
        print(f"[case] {what}: {name}", flush=True)
        got = ops.paged_attention_kv4(q, k, v, b.k_cache.shape[1], *b.meta(gpu), b.bs, b.scale, **kw)
        LC.check(got, *exact[some], f"{what}, {name}")


# ctx, new, q_heads, kv_heads, head_dim, block size
CASES = [
    ([1], [1], 4, 2, 64, 16),                                  # one key
    ([300], [1], 14, 2, 64, 256),                              # one token
    ([1500], [1], 28, 4, 128, 256),
    ([2000, 7, 65, 1, 640], [1] * 5, 28, 4, 128, 64),          # a ragged decode batch
    ([900, 128, 129], [1] * 3, 32, 8, 128, 16),                # eight kv heads, small blocks
    ([31, 32, 33, 16, 15, 17], [1] * 6, 8, 8, 64, 16),         # ends of 32 keys, one head a kv head
    ([700], [1], 16, 1, 128, 32),                              # 16 heads, one kv head
    ([700, 90], [1, 1], 40, 2, 128, 32),                       # 20 heads a kv head
    ([800, 90], [1, 1], 9, 3, 64, 48),                         # three kv heads
    ([300, 90], [1, 1], 12, 6, 128, 64),                       # six
    ([257, 64, 33], [257, 64, 33], 28, 4, 128, 64),            # packed prompts
    ([300], [300], 8, 8, 64, 16),
    ([333, 200], [120, 200], 14, 2, 64, 32),                   # a chunk after cached keys
    ([600, 31, 400], [40, 1, 3], 32, 8, 128, 256),             # decode tokens packed with chunks
    ([500, 90, 7], [5, 5, 5], 32, 8, 128, 64),                 # a few tokens of each sequence
    ([400, 90], [3, 2], 14, 2, 64, 16),
    ([90, 70], [90, 70], 6, 3, 96, 8),                         # other head and block sizes
    ([50, 40], [50, 2], 5, 1, 256, 24),
    ([45, 30], [45, 1], 3, 3, 32, 5),
    ([200, 60], [1, 1], 10, 2, 160, 16),
    ([200, 61], [4, 1], 8, 2, 256, 16),
    ([130] * 20, [1] * 20, 28, 4, 128, 64),                    # many sequences in a tile
    ([20, 140, 3, 64, 9], [20, 100, 2, 64, 9], 28, 4, 128, 16),
    ([1500, 900], [40, 21], 28, 4, 128, 64),                   # few tokens over many keys: key ranges
    ([1300], [33], 14, 2, 64, 16),
    ([120, 40], [2, 1], 130, 2, 64, 16),                       # 65 heads a kv head
    ([70] * 50 + [100, 90] + [20] * 30, [1] * 50 + [100, 60] + [1] * 30, 28, 4, 128, 32),  # over 64 sequences
]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ci", range(len(CASES)))
def test_kv4_attention(gpu, dt, ci):
    ctx, new, qh, kvh, hd, bs = CASES[ci]
    b, kc, vc = kv4.make_batch(ci, ctx, new, qh, kvh, hd, bs, dt)
    verify(gpu, b, kc, vc, f"case {ci}")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("hd,bs", [(64, 16), (128, 64), (96, 8)])
def test_key_counts(gpu, dt, hd, bs):
    """Padding rows, counts below zero, tokens that see less than their sequence holds: with junk behind."""
    ctx, new = [200, 90, 0, 40], [30, 1, 2, 8]
    n = np.concatenate([np.arange(171, 201), [90], [0, -(2 ** 31)], [40, 0, 1, -5, 17, 16, 15, 40]])
    b, kc, vc = kv4.make_batch(5, ctx, new, 8, 2, hd, bs, dt, key_len=n)
    verify(gpu, b, kc, vc, "key counts")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("hd,bs", [(128, 64), (64, 16), (32, 8)])
def test_keys_without_a_block(gpu, dt, hd, bs):
    """A seen key whose entry is no block, or whose sequence is no row of the tables: NaN; the other rows as before."""
    ctx, new = [300, 100, 80], [20, 1, 1]
    b, kc, vc = kv4.make_batch(6, ctx, new, 8, 2, hd, bs, dt)
    exact, tol = kv4.exact_attention(b, dt != torch.float32)
    b.table[1, 40 // bs] = 1 << 20
    lost = b.seq == 1
    b.seq = np.where(b.seq == 2, 7, b.seq)  # no row
    lost |= b.seq == 7
    q, k, v = b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    for kw in ({}, dict(cu_seqlens=b.cu), dict(split=False)):
        got = ops.paged_attention_kv4(q, k, v, 2, *b.meta(gpu), b.bs, b.scale, **kw)
        assert torch.isnan(got[torch.from_numpy(lost)]).all()
        LC.check(got[torch.from_numpy(~lost)], exact[~lost], tol[~lost], "others")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_groups_that_are_no_numbers(gpu, dt, hd):
    """A NaN group in K or V of one key: the tokens that see the key are NaN (of V: in those dimensions), earlier ones not."""
    ctx, new = [150, 60], [60, 1]
    b, kc, vc = kv4.make_batch(8, ctx, new, 8, 2, hd, 16, dt)
    exact, tol = kv4.exact_attention(b, dt != torch.float32)
    words = 2 * hd // 2
    rows = [b.table[0, j // 16] * 16 + j % 16 for j in (120, 130)]
    kc[rows[0], words:words + 2] = 0x00, 0x7E              # kv head 0, first group
    at = words + 2 * (hd // 32) + 2 * (hd // 32 - 1)
    vc[rows[1], at:at + 2] = 0x00, 0x7E                    # kv head 1, last group
    got = ops.paged_attention_kv4(b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), 2, *b.meta(gpu),
                                  16, b.scale).cpu()
    n = torch.from_numpy(b.key_len)
    want = torch.zeros(got.shape, dtype=torch.bool)
    first = torch.from_numpy(b.seq == 0)
    want[first & (n > 120), :4] = True
    want[(first & (n > 130))[:, None, None] & (torch.arange(8) >= 4)[:, None] & (torch.arange(hd) >= hd - 32)] = True
    assert torch.equal(torch.isnan(got), want)
    fine = ~want.numpy()
    assert (np.abs(got.double().numpy() - exact)[fine] <= tol[fine]).all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_scales_and_large_scores(gpu, dt):
    """Scales of zero and below it, scores in the hundreds, rows of q far apart in size and of zeros."""
    for ctx, new in (([300, 40], [20, 1]), ([300, 40], [1, 1])):
        b, kc, vc = kv4.make_batch(9, ctx, new, 8, 2, 128, 16, dt)
        for scale, size in ((0.0, 1.0), (-0.1, 1.0), (1.0, 8.0), (0.05, 1e-3), (1e-3, 1e3)):
            c = LC.dataclasses.replace(b, q=(b.q.float() * size).to(dt), scale=scale)
            c.q[0, 1] = 0
            c.q[-1, 2] = (c.q[-1, 2].float() * 2.0 ** -12).to(dt)
            verify(gpu, c, kc, vc, f"scale {scale}")


def test_strides_streams_and_graphs(gpu):
    """Rows of q with a gap, aligned and not; another stream; a captured call replayed on new inputs, next to eager calls."""
    dt, qh, kvh, hd, bs = torch.bfloat16, 28, 4, 128, 64
    b, kc, vc = kv4.make_batch(11, [700, 130, 1, 64], [1] * 4, qh, kvh, hd, bs, dt)
    exact, tol = kv4.exact_attention(b, False)
    k, v, meta = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), b.meta(gpu)
    for gap in (8, 3):
        wide = torch.zeros((4, qh * hd + gap), dtype=dt, device=gpu)
        wide[:, :qh * hd] = b.q.view(4, -1).to(gpu)
        q = wide[:, :qh * hd].unflatten(1, (qh, hd))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got = ops.paged_attention_kv4(q, k, v, kvh, *meta, bs, b.scale, max_query_len=1)
        stream.synchronize()
        LC.check(got, exact, tol, f"gap {gap}")
    q = b.q.to(gpu)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    ops.paged_attention_kv4(q, k, v, kvh, *meta, bs, b.scale, max_query_len=1, out=out)
    with torch.cuda.graph(graph):
        ops.paged_attention_kv4(q, k, v, kvh, *meta, bs, b.scale, max_query_len=1, out=out)
    for seed in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).to(dt))
        meta[1].copy_(torch.tensor([700 - 9 * seed, 130, 0 if seed == 2 else 1, 64 - seed], dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        eager = ops.paged_attention_kv4(q, k, v, kvh, *meta, bs, b.scale, max_query_len=1)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_one_token_over_a_cache_past_4_gib(gpu):
    """Blocks whose byte offsets pass 32 bits."""
    kvh, hd, bs, qh = 8, 128, 64, 32
    row = ops.kv4_row_bytes(kvh, hd)
    rows = ((5 << 30) // row) // bs * bs
    kc, vc = ops.kv4_cache(rows, kvh, hd, gpu), ops.kv4_cache(rows, kvh, hd, gpu)
    b, k, v = kv4.make_batch(12, [200], [1], qh, kvh, hd, bs, torch.float16)
    far = [rows // bs - 1 - i for i in range(4)]
    for i, page in enumerate(b.table[0, :4]):
        kc[far[i] * bs:(far[i] + 1) * bs] = torch.from_numpy(k[page * bs:(page + 1) * bs]).to(gpu)
        vc[far[i] * bs:(far[i] + 1) * bs] = torch.from_numpy(v[page * bs:(page + 1) * bs]).to(gpu)
    exact, tol = kv4.exact_attention(b, True)
    b.table[0, :4] = far
    meta = b.meta(gpu)
    for q, n in ((b.q, meta[1]),):
        for kw in (dict(max_query_len=1), {}):
            LC.check(ops.paged_attention_kv4(q.to(gpu), kc, vc, kvh, meta[0], n, meta[2], bs, b.scale, **kw), exact, tol, "far")
    # and tiles: forty tokens that all see the same keys
    many = b.q.to(gpu).expand(40, -1, -1).contiguous()
    got = ops.paged_attention_kv4(many, kc, vc, kvh, meta[0].expand(40).contiguous(), meta[1].expand(40).contiguous(),
                                  meta[2], bs, b.scale)
    LC.check(got, np.repeat(exact, 40, 0), np.repeat(tol, 40, 0), "far tiles")
