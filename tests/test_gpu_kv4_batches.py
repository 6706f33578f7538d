"""4-bit attention of batches past those whose keys are shared out: results, and that a larger batch, or one whose packing is given
in place of a promise, does not take another and much slower way."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC

pytestmark = pytest.mark.gpu


def args_of(gpu, b, kc, vc):
    return (b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), b.k_cache.shape[1], *b.meta(gpu), b.bs,
            b.scale)


# sequences' tokens, q_heads, kv_heads, head_dim
RAGGED = [(8, 4, 2, 64), (8, 4, 1, 64), (5, 8, 4, 128), (1, 14, 2, 64), (8, 4, 2, 256)]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("most,qh,kvh,hd", RAGGED)
def test_many_short_sequences(gpu, dt, most, qh, kvh, hd):
    """Some 1500 tokens of sequences of 0 to `most`, padding rows among them, with their packing and without."""
    r = np.random.default_rng(most)
    new = r.integers(0 if most > 1 else 1, most + 1, 3000 // (most + 1))
    ctx = np.maximum(r.integers(1, 60, len(new)), new)
    key_len = np.concatenate([np.arange(c - n, c) + 1 for c, n in zip(ctx, new)])
    key_len[::37] = 0
    b, kc, vc = kv4.make_batch(1, ctx, new, qh, kvh, hd, 16, dt, key_len=key_len)
    out, tol = kv4.exact_attention(b, dt != torch.float32)
    args = args_of(gpu, b, kc, vc)
    for kw in (dict(cu_seqlens=b.cu), dict(cu_seqlens=b.cu, split=False), dict(max_query_len=most), {}):
        LC.check(ops.paged_attention_kv4(*args, **kw), out, tol, str(kw))


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("tokens", [765, 770, 2045, 2050])
def test_both_sides_of_sharing(gpu, dt, tokens):
    """Short sequences, single tokens and tokens in any order."""
    for ctx, new in (([40] * (tokens // 10) + [9], [10] * (tokens // 10) + [tokens % 10]),
                     (np.arange(tokens) % 50 + 1, [1] * tokens)):
        b, kc, vc = kv4.make_batch(2, ctx, new, 4, 2, 256 if tokens < 1000 else 64, 16, dt)
        out, tol = kv4.exact_attention(b, dt != torch.float32)
        args = args_of(gpu, b, kc, vc)
        for kw in (dict(cu_seqlens=b.cu), {}):
            LC.check(ops.paged_attention_kv4(*args, **kw), out, tol, str(kw))
    at = np.random.default_rng(3).permutation(tokens)
    b.q, b.seq, b.key_len = b.q[torch.from_numpy(at)], b.seq[at], b.key_len[at]
    LC.check(ops.paged_attention_kv4(*args_of(gpu, b, kc, vc)), out[at], tol[at], "any order")


def test_capture(gpu):
    """A captured call of groups that are not shared out, replayed on other queries and key counts, eager calls between."""
    r = np.random.default_rng(4)
    new = r.integers(1, 6, 400)
    b, kc, vc = kv4.make_batch(4, np.maximum(r.integers(1, 90, 400), new), new, 8, 2, 128, 16, torch.bfloat16)
    q, k, v, kvh, seq, n, table, bs, scale = args_of(gpu, b, kc, vc)
    assert len(b.q) > 768
    out = torch.empty_like(q)
    call = lambda **kw: ops.paged_attention_kv4(q, k, v, kvh, seq, n, table, bs, scale, cu_seqlens=b.cu, **kw)
    call(out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out=out)
    first = n.clone()
    for seed in range(4):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).to(q.dtype))
        n.copy_(first if seed != 2 else torch.clamp(first - 3, min=0))
        out.fill_(float("nan"))
        graph.replay()
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def least_us(*calls) -> float:
    """The least time of the calls one after the other, of a few rounds of ten."""
    best = float("inf")
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(10):
            for f in calls:
                f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) * 100.0)
    return best


def call_of(gpu, ctx, new, qh, kvh, hd, bs, **kw):
    """A call over a cache of zeros (whose values do not matter for the time)."""
    ctx, new = np.asarray(ctx), np.asarray(new)
    pages = -(-ctx // bs)
    table = np.full((len(ctx), int(pages.max())), -1, np.int32)
    table[np.arange(table.shape[1]) < pages[:, None]] = np.arange(int(pages.sum()))
    seq = np.repeat(np.arange(len(ctx)), new).astype(np.int32)
    n = np.concatenate([np.arange(c - k, c) + 1 for c, k in zip(ctx, new)]).astype(np.int32)
    cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    k, v = (ops.kv4_cache(int(pages.sum()) * bs, kvh, hd, gpu) for _ in range(2))
    q = torch.ones((len(seq), qh, hd), dtype=torch.bfloat16, device=gpu)
    meta = [torch.from_numpy(x).to(gpu) for x in (seq, n, table)]
    return lambda: ops.paged_attention_kv4(q, k, v, kvh, *meta, bs, hd ** -0.5, cu_seqlens=cu, **kw)


def test_a_few_tokens_each_of_many_sequences(gpu):
    """128 sequences of 5 tokens take no longer than two calls of 64 (token by token they take twice as long)."""
    ctx = np.random.default_rng(5).integers(5, 4097, 128)
    whole = call_of(gpu, ctx, [5] * 128, 32, 8, 128, 64)
    parts = [call_of(gpu, c, [5] * 64, 32, 8, 128, 64) for c in (ctx[:64], ctx[64:])]
    a, b = least_us(whole), least_us(*parts)
    print(f"[perf] 128 sequences of 5 tokens {a:.0f} us, twice 64 {b:.0f}")
    assert a < 1.4 * b


def test_single_tokens_by_their_packing(gpu):
    """600 single tokens take no longer where the packing says so than where max_query_len does."""
    ctx = np.random.default_rng(6).integers(1, 4097, 600)
    packing, promise = (call_of(gpu, ctx, [1] * 600, 28, 4, 128, 64, **kw) for kw in ({}, dict(max_query_len=1)))
    a, b = least_us(packing), least_us(promise)
    print(f"[perf] 600 tokens {a:.0f} us by their packing, {b:.0f} promised")
    assert a < 1.2 * b


def test_a_bound_beside_the_packing(gpu):
    """A bound of the sequences' tokens beside their packing changes nothing."""
    ctx = np.random.default_rng(7).integers(5, 4097, 32)
    packing, both = (call_of(gpu, ctx, [5] * 32, 32, 8, 128, 64, **kw) for kw in ({}, dict(max_query_len=64)))
    a, b = least_us(packing), least_us(both)
    print(f"[perf] 32 sequences of 5 tokens {a:.0f} us by their packing, {b:.0f} with a bound")
    assert b < 1.3 * a


def test_chunks_of_head_size_256(gpu):
    """A chunk of 2060 tokens takes no longer than two of 1030."""
    whole = call_of(gpu, [4000], [2060], 16, 8, 256, 64)
    parts = [call_of(gpu, [c], [1030], 16, 8, 256, 64) for c in (2970, 4000)]
    a, b = least_us(whole), least_us(*parts)
    print(f"[perf] 2060 tokens {a:.0f} us, twice 1030 {b:.0f}")
    assert a < 1.25 * b
