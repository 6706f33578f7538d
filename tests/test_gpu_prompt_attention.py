"""Causal attention of packed prompts over their own rows, against its definition in 64 bits.

Tolerance: long_context.exact_attention's (fp32 sums, P rounded once to the storage type)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu


def exact(q, k, v, cu, scale):
    """(out, tolerance); rows of no sequence are zeros with no tolerance."""
    dt, (tokens, qh, hd) = q.dtype, q.shape
    kvh = k.shape[1]
    g = qh // kvh
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    q, k, v = (x.double().numpy() for x in (q, k, v))
    u = 2.0 ** -24
    for a, b in zip(cu, cu[1:]):
        for h in range(qh):
            kk, vv = k[a:b, h // g], v[a:b, h // g]
            for t in range(a, b):
                kt, vt = kk[:t - a + 1], vv[:t - a + 1]
                s = kt @ q[t, h] * scale
                p = np.exp(s - s.max())
                o = p @ vt / p.sum()
                S = abs(scale) * (np.abs(kt) @ np.abs(q[t, h])).max()
                n = t - a + 1
                e = 2 * (hd + 8) * u * S + (n + 8) * u
                if dt != torch.float32:
                    e += LC.half_step(dt)
                if dt == torch.float16:
                    e += n * 2.0 ** -25
                out[t, h] = o
                tol[t, h] = e * np.abs(vt).max() + LC.half_step(dt) * np.abs(o) + \
                    (2.0 ** -25 if dt == torch.float16 else 1e-30)
    return out, tol


def inputs(seed, tokens, qh, kvh, hd, dt):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((tokens, qh + 2 * kvh, hd), generator=g).to(dt)
    return qkv


def split_heads(qkv, qh, kvh):
    return qkv[:, :qh], qkv[:, qh:qh + kvh], qkv[:, qh + kvh:]


# lengths, q_heads, kv_heads, head_dim
CASES = [
    ([1], 4, 2, 64),
    ([2, 1, 1, 3], 14, 2, 64),
    ([37], 14, 2, 64),
    ([64, 65, 63], 28, 4, 128),          # ends of chunks
    ([18, 19, 17, 36], 28, 4, 128),      # ends of tiles
    ([200], 8, 8, 64),                   # one head a kv head
    ([130, 0, 150, 0], 32, 8, 128),      # empty sequences
    ([150], 16, 1, 128),
    ([70, 33], 40, 2, 128),              # 20 heads a kv head
    ([60, 33], 130, 2, 64),              # 65
    ([90, 1, 44], 6, 3, 80),             # other head sizes
    ([50, 40], 5, 1, 256),
    ([45], 3, 3, 37),
    ([9] * 40 + [1] * 50, 28, 4, 128),   # many short sequences: over 64
    ([400], 14, 2, 64),
    ([], 4, 2, 64),                      # no sequence at all
]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ci", range(len(CASES)))
def test_prompt_attention(gpu, dt, ci):
    lens, qh, kvh, hd = CASES[ci]
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    tokens = int(cu[-1]) + 5  # rows behind the last sequence
    qkv = inputs(ci, tokens, qh, kvh, hd, dt)
    qkv[int(cu[-1]):] = float("nan")
    q, k, v = split_heads(qkv, qh, kvh)
    want, tol = exact(q, k, v, cu.tolist(), hd ** -0.5)
    d = split_heads(qkv.to(gpu), qh, kvh)
    dcu = torch.from_numpy(cu).to(gpu)
    for name, rows, split in (("packed rows", d, True), ("contiguous", [x.contiguous() for x in d], True),
                              ("unsplit", d, False)):
        print(f"[case] {ci}: {name}", flush=True)
        out = torch.full((tokens, qh, hd), 7.0, dtype=dt, device=gpu)
        assert ops.prompt_attention(*rows, dcu, hd ** -0.5, out=out, split=split) is out
        LC.check(out[:int(cu[-1])], want[:int(cu[-1])], tol[:int(cu[-1])], name)
        assert (out[int(cu[-1]):] == 7).all(), "rows behind the last sequence"


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("hd", [64, 128, 48])
def test_masked_rows_hold_anything(gpu, dt, hd):
    """Infinities and NaN in later keys and values, and in the sequences beside: earlier rows are as without them."""
    qh, kvh, lens = 14, 2, [40, 90, 30]
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    qkv = inputs(3, 160, qh, kvh, hd, dt)
    q, k, v = split_heads(qkv, qh, kvh)
    want, tol = exact(q, k, v, cu.tolist(), hd ** -0.5)
    k[cu[1] + 70, 0, 3], v[cu[1] + 60, 1, 5] = float("nan"), float("inf")
    k[130:], v[130:] = float("inf"), float("nan")
    got = ops.prompt_attention(*split_heads(qkv.to(gpu), qh, kvh), torch.from_numpy(cu).to(gpu), hd ** -0.5)
    fine = np.ones(want.shape, bool)
    fine[130:] = False
    fine[cu[1] + 70:130, :7] = False
    fine[cu[1] + 60:130, 7:, 5] = False
    g = got.double().cpu().numpy()
    assert (np.abs(g - want)[fine] <= tol[fine]).all()
    assert np.isnan(g[cu[1] + 70:130, :7]).all() and (~np.isfinite(g[cu[1] + 60:130, 7:, 5])).all()


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_first_token_offset_and_odd_rows(gpu, dt):
    """A packing that begins behind the first row, rows that are not 16-byte aligned, strides of K and V apart, scales of zero and
    below."""
    qh, kvh, hd, cu = 6, 2, 64, [7, 60, 61, 130]
    for scale in (hd ** -0.5, 0.0, -0.2):
        qkv = inputs(4, 140, qh, kvh, hd, dt)
        q, k, v = split_heads(qkv, qh, kvh)
        want, tol = exact(q, k, v, cu, scale)
        wide = torch.zeros((140, kvh * hd + 5), dtype=dt, device=gpu)
        wide[:, 5:] = v.reshape(140, -1).to(gpu)
        even = torch.zeros((140, kvh * hd + 64), dtype=dt, device=gpu)
        even[:, 64:] = v.reshape(140, -1).to(gpu)
        for vd in (wide[:, 5:].unflatten(1, (kvh, hd)), even[:, 64:].unflatten(1, (kvh, hd))):
            out = torch.full((140, qh, hd), -3.0, dtype=dt, device=gpu)
            ops.prompt_attention(q.to(gpu), k.to(gpu), vd, torch.tensor(cu, dtype=torch.int32, device=gpu), scale, out=out)
            LC.check(out[7:130], want[7:130], tol[7:130], f"scale {scale}")
            assert (out[:7] == -3).all() and (out[130:] == -3).all()


@pytest.mark.parametrize("hd", [128, 80])
def test_packings_outside_the_rows(gpu, hd):
    """Entries below zero, past the tokens and decreasing ones: the rows stay within the arrays, right where a sequence is one."""
    dt, qh, kvh = torch.float16, 4, 2
    qkv = inputs(5, 100, qh, kvh, hd, dt).to(gpu)
    guard = torch.full((300, qh, hd), 5.0, dtype=dt, device=gpu)
    for cu in ([-40, 50, 1 << 30], [0, 90, 20, 100], [2 ** 31 - 1, -(2 ** 31)], [50, 50, 50], [100, 200], [-9, -3]):
        guard.fill_(5.0)
        ops.prompt_attention(*split_heads(qkv, qh, kvh), torch.tensor(cu, dtype=torch.int32, device=gpu), hd ** -0.5,
                             out=guard[100:200])
        assert (guard[:100] == 5).all() and (guard[200:] == 5).all(), cu
    want, tol = exact(*split_heads(qkv.cpu(), qh, kvh), [0, 50, 100], hd ** -0.5)
    out = ops.prompt_attention(*split_heads(qkv, qh, kvh), torch.tensor([-40, 50, 1 << 30], dtype=torch.int32, device=gpu),
                               hd ** -0.5)
    LC.check(out, want, tol, "bounds")


def test_streams_and_graphs(gpu):
    """Another stream, and a captured call replayed on other rows and another packing, with eager calls between."""
    dt, qh, kvh, hd, tokens = torch.bfloat16, 28, 4, 128, 300
    qkv = inputs(6, tokens, qh, kvh, hd, dt).to(gpu)
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device=gpu)
    out = torch.zeros((tokens, qh, hd), dtype=dt, device=gpu)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.prompt_attention(*split_heads(qkv, qh, kvh), cu, hd ** -0.5, out=out)
    stream.synchronize()
    assert torch.equal(out[:290], ops.prompt_attention(*split_heads(qkv, qh, kvh), cu, hd ** -0.5)[:290])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.prompt_attention(*split_heads(qkv, qh, kvh), cu, hd ** -0.5, out=out)
    for seed, packing in enumerate(([0, 100, 290], [0, 1, 300], [0, 0, 0], [10, 20, 280])):
        qkv.copy_(inputs(seed, tokens, qh, kvh, hd, dt))
        cu.copy_(torch.tensor(packing, dtype=torch.int32))
        out.fill_(2.0)
        graph.replay()
        eager = torch.full_like(out, 2.0)
        ops.prompt_attention(*split_heads(qkv, qh, kvh), cu, hd ** -0.5, out=eager)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
