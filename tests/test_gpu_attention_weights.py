"""The softmax weights of window and prefix attention over 16-bit caches, held as two 16-bit parts.

The tolerance is long_context.exact_attention's without its half step of the type for P: one part is off by half a
step of the type relatively, so the second, which holds what the first left, by half a step of half a step:
2^-8 * 2^-8 in bf16, 2^-11 * 2^-11 in fp16, there or by half of the least subnormal, 2^-25 for each key (the
largest weight of a row is at least 1, and so is their sum)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu

DTYPES = LC.DTYPES[1:]
IDS = LC.DT_IDS[1:]


def exact_weights(b, window=1 << 30, sinks=0):
    """(out, tolerance) in 64 bits, for weights in two parts."""
    out, tol = LC.exact_attention(b, window, sinks)
    step = LC.half_step(b.q.dtype)
    kv_heads = b.k_cache.shape[1]
    v = b.v_cache.double().abs().numpy()
    for t in range(len(b.seq)):
        j = np.flatnonzero(LC.seen_keys(int(b.key_len[t]), window, sinks))
        if len(j):
            rows = b.table[b.seq[t], j // b.bs] * b.bs + j % b.bs
            group = b.q.shape[1] // kv_heads
            for h in range(kv_heads):
                tol[t, h * group:(h + 1) * group] -= (step - step * step) * v[rows, h].max()
    return out, tol


# ctx (one token each), q_heads, kv_heads, head_dim, block size, window, sinks
DECODE = [
    ([700], 28, 4, 128, 64, 1 << 20, 0),
    ([3000, 7, 65, 1, 640], 28, 4, 128, 64, 512, 4),
    ([1500], 14, 2, 64, 256, 1000, 70),
    ([900, 128, 129], 32, 8, 128, 16, 64, 1),
    ([700, 90], 40, 2, 128, 32, 100, 3),
    ([400, 33], 16, 1, 64, 16, 300, 0),
]


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("ci", range(len(DECODE)))
def test_single_tokens(gpu, dt, ci):
    """Keys in one range and in several: both are near the exact result, so near each other."""
    ctx, qh, kvh, hd, bs, window, sinks = DECODE[ci]
    b = LC.make_batch(300 + ci, ctx, [1] * len(ctx), qh, kvh, hd, bs, dt, window, sinks)
    exact, tol = exact_weights(b, window, sinks)
    d, meta = b.to(gpu), b.meta(gpu)
    for split in (True, False):
        got = ops.window_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, window, sinks, max_query_len=1,
                                   split=split)
        LC.check(got, exact, tol, f"split={split}")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_own_keys_of_a_prefix_call(gpu, dt, hd):
    b = LC.make_batch(320, [400, 90, 33, 1000], [1] * 4, 28, 4, hd, 64, dt)
    exact, tol = exact_weights(b)
    d, meta = b.to(gpu), b.meta(gpu)
    LC.check(ops.prefix_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 0), exact, tol, "no prefix")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_shared_prefix(gpu, dt, hd):
    """A prefix read once for its tokens, and by each for itself."""
    b = LC.make_batch(331, [700], [40], 14, 2, hd, 16, dt)
    exact, tol = exact_weights(b)
    d, meta = b.to(gpu), b.meta(gpu)
    for share in (True, False):
        LC.check(ops.prefix_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 600, share=share), exact, tol,
                 f"share={share}")


@pytest.mark.parametrize("dt", DTYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("value", [float("inf"), -float("inf")])
def test_infinite_values(gpu, dt, hd, value):
    """An infinite value of a seen key is the result in its dimension, whatever sign a weight's second part has;
    a large finite one stays finite."""
    b = LC.make_batch(332, [90, 65], [1, 1], 14, 2, hd, 16, dt)
    for s, key in ((0, 31), (1, 64)):
        row = int(b.table[s, key // 16]) * 16 + key % 16
        b.v_cache[row, :, 5] = value
    b.v_cache[int(b.table[0, 2]) * 16 + 3, :, 9] = min(torch.finfo(dt).max, 2.0 ** 100)
    d, meta = b.to(gpu), b.meta(gpu)
    for got in (ops.window_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 1 << 20, max_query_len=1),
                ops.window_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 1 << 20, max_query_len=1, split=False),
                ops.prefix_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 0)):
        assert (got[:, :, 5] == value).all()
        rest = torch.cat([got[:, :, :5], got[:, :, 6:]], 2)
        assert torch.isfinite(rest).all()
