"""4-bit attention where it can go wrong beside test_gpu_kv4_attention's shapes: values that fp16 holds as subnormals, large
ones, batches past those that are shared out, tokens in any order, calls at once on two streams and two captured graphs."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC

pytestmark = pytest.mark.gpu


def on(gpu, b, kc, vc, **kw):
    return ops.paged_attention_kv4(b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), b.k_cache.shape[1],
                                   *b.meta(gpu), b.bs, b.scale, **kw)


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("size", [1e-6, 1e-4, 60.0, 9000.0])
@pytest.mark.parametrize("new", [[1, 1], [5, 3], [60, 20]], ids=["single", "few", "chunk"])
def test_small_and_large_values(gpu, dt, size, new):
    """K and V of one size, q such that scores are ordinary (or all near zero)."""
    qh, kvh, hd, bs = 8, 2, 128, 16
    g = torch.Generator().manual_seed(2)
    b, _, _ = kv4.make_batch(21, [150, 70], new, qh, kvh, hd, bs, dt)
    rows = b.k_cache.shape[0]
    kc, vc = (kv4.pack(*kv4.quantize((torch.randn((rows, kvh, hd), generator=g) * size).double().numpy())) for _ in range(2))
    b.k_cache, b.v_cache = (torch.from_numpy(kv4.values(c, kvh, hd)) for c in (kc, vc))
    b.scale = hd ** -0.5 / max(size, 1.0)
    for kw in (dict(cu_seqlens=b.cu), {}):
        some = dt != torch.float32 and len(b.q) * (qh // kvh) > 16
        out, tol = kv4.exact_attention(b, some)
        got = on(gpu, b, kc, vc, **kw)
        if dt == torch.float16:  # (past its largest number)
            fine = torch.from_numpy(np.abs(out) < 60000)
            got, out, tol = torch.where(fine, got.cpu(), 0), np.where(fine, out, 0), np.where(fine, tol, 0)
        LC.check(got, out, tol, f"size {size}")


@pytest.mark.parametrize("dt", [torch.float16, torch.float32], ids=["f16", "f32"])
def test_large_batches(gpu, dt):
    """More single tokens than are shared out, and as many as are."""
    for tokens in (2048, 2100):
        r = np.random.default_rng(tokens)
        ctx = r.integers(1, 50, tokens)
        b, kc, vc = kv4.make_batch(22, ctx, [1] * tokens, 4, 2, 64, 16, dt)
        LC.check(on(gpu, b, kc, vc, max_query_len=1), *kv4.exact_attention(b, False), f"{tokens} tokens")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("qh,kvh,hd", [(14, 2, 64), (32, 8, 128), (6, 6, 128), (4, 1, 256)])
def test_tokens_in_any_order(gpu, dt, qh, kvh, hd):
    """Tokens of a sequence apart from each other and out of order, with every promise that holds."""
    b, kc, vc = kv4.make_batch(23, [90, 130, 40, 65], [5, 30, 2, 3], qh, kvh, hd, 16, dt)
    at = np.random.default_rng(1).permutation(len(b.seq))
    b.q, b.seq, b.key_len = b.q[torch.from_numpy(at)], b.seq[at], b.key_len[at]
    out, tol = kv4.exact_attention(b, dt != torch.float32)
    for kw in ({}, dict(max_query_len=30), dict(max_query_len=2), dict(max_query_len=1), dict(split=False)):
        LC.check(on(gpu, b, kc, vc, **kw), out, tol, str(kw))


def test_calls_at_once(gpu):
    """Two streams with calls of their own in flight, and two captured graphs replayed in turn: no workspace is shared."""
    dt, kvh, hd, bs = torch.bfloat16, 4, 128, 64
    batches = []
    for seed, new in ((31, [1] * 6), (32, [4, 6, 3, 2, 5, 1])):
        b, kc, vc = kv4.make_batch(seed, [900, 64, 300, 31, 500, 7], new, 28, kvh, hd, bs, dt)
        args = (b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), kvh, *b.meta(gpu), bs, b.scale)
        kw = dict(cu_seqlens=b.cu)
        batches.append((args, kw, ops.paged_attention_kv4(*args, **kw), kv4.exact_attention(b, True)))
    for _, _, got, (out, tol) in batches:
        LC.check(got, out, tol, "alone")
    streams = [torch.cuda.Stream() for _ in batches]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(10):
        for i, (args, kw, _, _) in enumerate(batches):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_attention_kv4(*args, **kw))
    torch.cuda.synchronize()
    for i, (_, _, want, _) in enumerate(batches):
        assert all(torch.equal(g, want) for g in got[i])
    graphs, outs = [], []
    for args, kw, _, _ in batches:
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(args[0])
        with torch.cuda.graph(graph):
            ops.paged_attention_kv4(*args, **kw, out=out)
        graphs.append(graph)
        outs.append(out)
    for _ in range(3):
        for out in outs:
            out.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for out, (_, _, want, _) in zip(outs, batches):
            assert torch.equal(out, want)


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_prompt_and_cache_agree(gpu, dt):
    """prompt_attention over what a 4-bit cache gives back is paged_attention_kv4 over the cache, to rounding."""
    qh, kvh, hd, bs, n = 8, 2, 64, 16, 120
    b, kc, vc = kv4.make_batch(24, [n], [n], qh, kvh, hd, bs, dt)
    k, v = (ops.kv4_unpack(torch.from_numpy(c).to(gpu), kvh, hd, torch.float32) for c in (kc, vc))
    rows = torch.from_numpy(b.table[0, np.arange(n) // bs] * bs + np.arange(n) % bs).to(gpu)
    out, tol = kv4.exact_attention(b, dt != torch.float32)
    LC.check(on(gpu, b, kc, vc, cu_seqlens=b.cu), out, tol, "cache")
    if dt == torch.float32:  # (16-bit rows would round the values)
        got = ops.prompt_attention(b.q.to(gpu), k[rows], v[rows], torch.tensor([0, n], dtype=torch.int32, device=gpu), b.scale)
        LC.check(got, out, tol, "prompt")


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("qh,kvh,hd", [(8, 2, 64), (8, 4, 128), (6, 1, 128), (16, 8, 64), (4, 2, 256)])
def test_a_few_tokens_and_groups_that_are_no_numbers(gpu, dt, qh, kvh, hd):
    """A NaN group in K and one in V of keys that only the later ones of a few tokens see: the earlier ones are as without."""
    ctx, new, bs = [150, 90], [3, 2], 16
    b, kc, vc = kv4.make_batch(25, ctx, new, qh, kvh, hd, bs, dt)
    out, tol = kv4.exact_attention(b, dt != torch.float32)
    words, of_head = kvh * hd // 2, 2 * (hd // 32)
    at = [b.table[s, (n - 1) // bs] * bs + (n - 1) % bs for s, n in enumerate(ctx)]
    kc[at[0], words:words + 2] = 0x00, 0x7E                                   # kv head 0, first group
    last = words + kvh * of_head - 2
    vc[at[1], last:last + 2] = 0x00, 0x7E                                     # last kv head, last group
    want = np.zeros(out.shape, bool)
    g = qh // kvh
    want[2, :g] = True                  # the first sequence's last token, kv head 0
    want[4, qh - g:, hd - 32:] = True   # the second one's, last kv head, last 32 dimensions
    for kw in (dict(cu_seqlens=b.cu), {}, dict(cu_seqlens=b.cu, split=False)):
        got = on(gpu, b, kc, vc, **kw).double().cpu().numpy()
        assert np.array_equal(np.isnan(got), want), kw
        assert (np.abs(got - out)[~want] <= tol[~want]).all(), kw


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("n", [2, 3, 5, 7])
def test_sequences_of_as_many_tokens(gpu, dt, n):
    """The tokens that share columns end where sequences of n tokens do, where n is known, and anywhere where it is not."""
    ctx = [400, 33, n, 129, 70, 257, 64]
    b, kc, vc = kv4.make_batch(26, ctx, [n] * len(ctx), 8, 4, 128, 16, dt)
    out, tol = kv4.exact_attention(b, dt != torch.float32)
    for kw in (dict(cu_seqlens=b.cu), dict(max_query_len=n), dict(max_query_len=n, split=False), {}):
        LC.check(on(gpu, b, kc, vc, **kw), out, tol, str(kw))
