"""Small softmax weights: a key some 17 nats ahead of thousands of others, whose own value is zero, so that the output is
what the small weights make of it.  A weight below half of fp16's least subnormal must not be lost, nor one near it
keep a few bits only.

q is one number a head (its other dimensions are zero), so a score is one product and the tolerance stays narrow."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def floor(dt):
    """What a weight as fp16 numbers may lose, the row's largest weight being 1."""
    return 2.0 ** -38 if dt == torch.float32 else 2.0 ** -32


def row(s, v, scale, rel, least, dt):
    """(out, tolerance) of one (token, head) with products s = q . k (exact in fp32) over values v [n, hd], in 64 bits.

      exponents: score times scale times log2(e), less the reference: three roundings of numbers of at most x = |scale s| log2(e)
                 + 16 and one of the exponential, so 4 u x + 2 u of p; it moves p in both sums;
      weights:   rel of itself (but never more than all of it) and `least` of the largest;
      sums:      n + 8 roundings of the sum of p |V| and of the sum of p;
      out:       half a step of the type, of its own value."""
    x = s * scale
    p = np.exp(x - x.max())
    o = p @ v / p.sum()
    n = len(s)
    moved = p * (4 * U * (np.abs(x).max() * 1.4427 + 16) + 2 * U)
    lost = np.minimum(p, rel * p + least)
    e = (moved @ (np.abs(v) + np.abs(o)) + lost @ np.abs(v)) / p.sum() + 2 * (n + 8) * U * (p @ np.abs(v)) / p.sum()
    return o, e * 1.001 + LC.half_step(dt) * np.abs(o) + (2.0 ** -25 if dt == torch.float16 else 1e-30)


def values(r, n, ahead, spread, last):
    """The keys' one number and the values [n, hd] of a sequence."""
    k = r.uniform(-spread, spread, n) if spread else np.zeros(n)
    first = n - 1 if last else 0
    k[first] = ahead
    v = r.normal(2.0, 0.5, (n, 1))
    v[first] = 0.0
    return k, v


def batch(seed, ctx, new, qh, kvh, hd, bs, dt, ahead, spread, last):
    """(long_context.Batch, K rows, V rows) of such sequences."""
    b, _, _ = kv4.make_batch(seed, ctx, new, qh, kvh, hd, bs, dt)
    r = np.random.default_rng(seed)
    k, v = np.zeros((2, b.k_cache.shape[0], kvh, hd))
    for s, n in enumerate(ctx):
        j = np.arange(n)
        rows = b.table[s, j // bs] * bs + j % bs
        for h in range(kvh):
            kk, vv = values(r, n, ahead, spread, last)
            k[rows, h, 0] = kk
            v[rows, h] = vv * r.uniform(0.5, 1.5, (1, hd)) * (vv > 0)
    kc, vc = kv4.pack(*kv4.quantize(k)), kv4.pack(*kv4.quantize(v))
    b.k_cache, b.v_cache = (torch.from_numpy(kv4.values(c, kvh, hd)) for c in (kc, vc))
    b.q.zero_()
    b.q[:, :, 0] = 8.0
    b.scale = 0.125
    return b, kc, vc


def exact(b, rel):
    out, tol = np.zeros(b.q.shape), np.zeros(b.q.shape)
    group = b.q.shape[1] // b.k_cache.shape[1]
    k, v, q = b.k_cache.numpy(), b.v_cache.numpy(), b.q.double().numpy()
    for t in range(len(b.seq)):
        j = np.arange(int(b.key_len[t]))
        rows = b.table[b.seq[t], j // b.bs] * b.bs + j % b.bs
        for h in range(q.shape[1]):
            out[t, h], tol[t, h] = row(k[rows, h // group, 0] * q[t, h, 0], v[rows, h // group], b.scale, rel, floor(b.q.dtype),
                                         b.q.dtype)
    return out, tol


# how far ahead, in nats, the others' spread
TAILS = [(17.7, 0.0), (17.0, 3.0), (14.1, 0.0), (23.0, 0.0)]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ahead,spread", TAILS)
@pytest.mark.parametrize("qh,kvh,hd", [(14, 2, 64), (8, 4, 128), (8, 8, 128), (4, 1, 256), (4, 2, 96)])
@pytest.mark.parametrize("last", [False, True], ids=["first", "last"])
def test_single_tokens(gpu, dt, ahead, spread, qh, kvh, hd, last):
    b, kc, vc = batch(1, [3000, 700], [1, 1], qh, kvh, hd, 16 if hd != 96 else 8, dt, ahead, spread, last)
    out, tol = exact(b, 2.0 ** -22)
    args = (b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), kvh, *b.meta(gpu), b.bs, b.scale)
    for kw in (dict(max_query_len=1), dict(max_query_len=1, split=False), dict(cu_seqlens=b.cu)):
        LC.check(ops.paged_attention_kv4(*args, **kw), out, tol, str(kw))


@pytest.mark.parametrize("qh,kvh,hd", [(14, 2, 64), (8, 8, 128), (4, 1, 256), (4, 2, 96)])
@pytest.mark.parametrize("new", [[1, 1, 1], [4, 2, 3], [30, 7, 20]], ids=["single", "few", "chunk"])
def test_ordinary_weights(gpu, qh, kvh, hd, new):
    """Few keys of weights near each other in fp32, whose tolerance is below what one fp16 number for a weight would cost; in
    order, and with the tokens in any order."""
    b, kc, vc = batch(4, [40, 7, 65], new, qh, kvh, hd, 16 if hd != 96 else 8, torch.float32, 1.0, 3.0, False)
    out, tol = exact(b, 2.0 ** -22)
    at = np.random.default_rng(5).permutation(len(b.q))
    for order in (np.arange(len(b.q)), at):
        q, (seq, n, table) = b.q.to(gpu)[torch.from_numpy(order).to(gpu)], b.meta(gpu)
        where = torch.from_numpy(order).to(gpu)
        args = (q, torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), kvh, seq[where], n[where], table, b.bs, b.scale)
        for kw in ({}, dict(split=False), dict(max_query_len=1)):
            LC.check(ops.paged_attention_kv4(*args, **kw), out[order], tol[order], str(kw))


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ahead,spread", TAILS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [[4, 3], [40, 33]], ids=["few", "chunk"])
def test_several_tokens(gpu, dt, ahead, spread, hd, new):
    """(16-bit types: their calls may round a weight once to fp16.)"""
    b, kc, vc = batch(2, [2000, 300], new, 8, 2, hd, 16, dt, ahead, spread, False)
    out, tol = exact(b, 2.0 ** -22 if dt == torch.float32 else 2.0 ** -11)
    args = (b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), 2, *b.meta(gpu), b.bs, b.scale)
    for kw in (dict(cu_seqlens=b.cu), {}, dict(split=False)):
        LC.check(ops.paged_attention_kv4(*args, **kw), out, tol, str(kw))


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ahead,spread", TAILS)
@pytest.mark.parametrize("hd", [64, 128, 80])
def test_prompts(gpu, dt, ahead, spread, hd):
    """The first row of each prompt ahead of the rest.  (bf16 weights have fp32's exponents: no floor.)"""
    qh, kvh, lens, scale = 4, 2, [900, 130], 0.125
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    r = np.random.default_rng(3)
    q, k, v = np.zeros((cu[-1], qh, hd)), np.zeros((cu[-1], kvh, hd)), np.zeros((cu[-1], kvh, hd))
    q[:, :, 0] = 8.0
    for a, n in zip(cu, lens):
        for h in range(kvh):
            kk, vv = values(r, n, ahead, spread, False)
            k[a:a + n, h, 0] = kk
            v[a:a + n, h] = vv * r.uniform(0.5, 1.5, (1, hd))
    q, k, v = (torch.from_numpy(x).to(dt) for x in (q, k, v))
    got = ops.prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), torch.from_numpy(cu).to(gpu), scale)
    rel = 0.0 if dt == torch.float32 else LC.half_step(dt)
    qn, kn, vn = (x.double().numpy() for x in (q, k, v))
    out, tol = np.zeros(got.shape), np.zeros(got.shape)
    for a, n in zip(cu, lens):
        for t in range(a, a + n):
            for h in range(qh):
                out[t, h], tol[t, h] = row(kn[a:t + 1, h // 2, 0] * qn[t, h, 0], vn[a:t + 1, h // 2], scale, rel,
                                           floor(dt) if dt == torch.float16 else 0.0, dt)
    LC.check(got, out, tol, "prompt")
