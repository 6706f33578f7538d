"""Rotary positions (half and interleaved pairs, part of the head, scaled, far positions) and the store.

Tolerance: with u = half a step of fp32 (2^-24) and y = s (a cos - b sin), |y| <= s (|a| + |b|):
  cos and sin: 2^-52 |angle| from the fp64 product and reduction, u |r| <= pi u for rounding the
      reduced angle to fp32, and 2 units of the fp32 functions (documented maxima: 1 to 2 ulp), 4 u in all;
  the products, the sum and the scale: 4 u;
  the norm (where asked): hd + 8 roundings of the sum of squares, halved by the root, and 4 products;
  the store: half a step of the type."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def inputs(seed, tokens, qh, kvh, hd, rot, dt, far, norm):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn((tokens, (qh + 2 * kvh) * hd), generator=g).to(dt)
    positions = torch.randint(0, far, (tokens,), generator=g)
    if tokens > 3:
        positions[0], positions[1], positions[2] = 0, far, -5
    inv_freq, _ = ops.rotary_inv_freq(1e6, rot) if rot else (torch.zeros(0, dtype=torch.float64), 1.0)
    w = [(1 + 0.1 * torch.randn((hd,), generator=g)).to(dt) if norm else None for _ in range(2)]
    return qkv, positions, inv_freq, w


def exact(qkv, positions, inv_freq, w, qh, kvh, hd, interleaved, scale, dt):
    """(q, k, tolerances) in 64 bits."""
    tokens, rot = qkv.shape[0], 2 * len(inv_freq)
    x = qkv[:, :(qh + kvh) * hd].double().numpy().reshape(tokens, qh + kvh, hd).copy()
    rel = 0.0
    if w[0] is not None:
        x /= np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)
        x[:, :qh] *= w[0].double().numpy()
        x[:, qh:] *= w[1].double().numpy()
        rel = ((hd + 8) / 2 + 4) * U
    angle = positions.double().numpy()[:, None] * inv_freq.numpy()
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else \
        (np.arange(rot // 2), np.arange(rot // 2) + rot // 2)
    y, tol = x.copy(), np.abs(x) * rel
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = scale * (a * cos - b * sin), scale * (b * cos + a * sin)
    e = scale * (np.abs(a) + np.abs(b)) * (rel + (np.pi + 4 + 4) * U + 2.0 ** -52 * np.abs(angle)[:, None])
    tol[..., ia], tol[..., ib] = e, e
    tol += np.abs(y) * LC.half_step(dt) + (2.0 ** -25 if dt == torch.float16 else 1e-30)
    return y[:, :qh].reshape(tokens, -1), y[:, qh:].reshape(tokens, -1), \
        tol[:, :qh].reshape(tokens, -1), tol[:, qh:].reshape(tokens, -1)


# tokens, q_heads, kv_heads, head_dim, rotary_dim
SHAPES = [(1, 14, 2, 64, 64), (37, 28, 4, 128, 128), (300, 32, 8, 128, 64), (5, 3, 1, 256, 256), (9, 6, 3, 80, 32),
          (4, 5, 5, 37, 10), (33, 14, 2, 64, 32), (7, 2, 2, 128, 96), (3, 1, 1, 2, 2), (6, 4, 2, 128, 0),
          (21, 100, 3, 64, 16), (2, 4, 4, 256, 8)]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
@pytest.mark.parametrize("ci", range(len(SHAPES)))
def test_rotary(gpu, dt, interleaved, norm, ci):
    tokens, qh, kvh, hd, rot = SHAPES[ci]
    qn, kn = qh * hd, kvh * hd
    qkv, positions, inv_freq, w = inputs(ci, tokens, qh, kvh, hd, rot, dt, 1_000_000, norm)
    scale = 1.25 if ci % 2 else 1.0
    q, k, tq, tk = exact(qkv, positions, inv_freq, w, qh, kvh, hd, interleaved, scale, dt)
    d, p, f = qkv.to(gpu), positions.to(gpu), inv_freq.to(gpu)
    wd = [x.to(gpu) if x is not None else None for x in w]
    kw = dict(interleaved=interleaved, attn_scale=scale, q_w=wd[0], k_w=wd[1])
    print(f"[case] {SHAPES[ci]} {dt}", flush=True)
    qo, ko = torch.empty(tokens, qn, dtype=dt, device=gpu), torch.empty(tokens, kn, dtype=dt, device=gpu)
    ops.rotary(d[:, :qn], d[:, qn:qn + kn], p, f, qh, kvh, hd, q_out=qo, k_out=ko, **kw)
    LC.check(qo, q, tq, "q")
    LC.check(ko, k, tk, "k")
    assert torch.equal(d.cpu(), qkv)  # the inputs are left
    # stored: rows outside the cache and below zero are not
    rows = tokens + 5
    slots = torch.from_numpy(np.random.default_rng(ci).permutation(rows)[:tokens].astype(np.int32))
    if tokens > 3:
        slots[1], slots[2] = -1, rows
    kc, vc = (torch.full((rows, kvh, hd), 7.0, dtype=dt, device=gpu) for _ in range(2))
    qs = torch.empty_like(qo)
    ops.rotary_store_kv(d[:, :qn], d[:, qn:qn + kn], d[:, qn + kn:], p, f, qh, kvh, hd, kc, vc, slots.to(gpu), q_out=qs,
                        **kw)
    assert torch.equal(qs, qo) and torch.equal(d.cpu(), qkv)
    wk, wv = (torch.full((rows, kvh, hd), 7.0, dtype=dt) for _ in range(2))
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < rows:
            wk[s], wv[s] = ko[t].cpu().view(kvh, hd), qkv[t, qn + kn:].view(kvh, hd)
    assert torch.equal(kc.cpu(), wk) and torch.equal(vc.cpu(), wv)
    # in place, in a packed row, on another stream
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        e = d.clone()
        ops.rotary(e[:, :qn], e[:, qn:qn + kn], p, f, qh, kvh, hd, **kw)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(e[:, :qn], qo) and torch.equal(e[:, qn:qn + kn], ko)
    assert torch.equal(e[:, qn + kn:].cpu(), qkv[:, qn + kn:])
    # with the rotated k kept beside the cache
    e = d.clone()
    kc2 = torch.full_like(kc, 7.0)
    ops.rotary_store_kv(e[:, :qn], e[:, qn:qn + kn], e[:, qn + kn:], p, f, qh, kvh, hd, kc2, torch.empty_like(vc),
                        slots.to(gpu), k_out=e[:, qn:qn + kn], **kw)
    assert torch.equal(e[:, :qn], qo) and torch.equal(e[:, qn:qn + kn], ko) and torch.equal(kc2, kc)


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_unaligned_rows(gpu, dt, interleaved):
    qkv, positions, inv_freq, w = inputs(50, 11, 4, 2, 64, 64, dt, 5000, False)
    q, k, tq, tk = exact(qkv, positions, inv_freq, w, 4, 2, 64, interleaved, 1.0, dt)
    rows = torch.zeros(11, 513, dtype=dt, device=gpu)
    rows[:, 1:] = qkv.to(gpu)
    ops.rotary(rows[:, 1:257], rows[:, 257:385], positions.to(gpu), inv_freq.to(gpu), 4, 2, 64, interleaved=interleaved)
    LC.check(rows[:, 1:257], q, tq, "q")
    LC.check(rows[:, 257:385], k, tk, "k")
    assert not rows[:, 0].any() and torch.equal(rows[:, 385:].cpu(), qkv[:, 384:])


def test_q_alone_and_no_tokens(gpu):
    qkv, positions, inv_freq, w = inputs(51, 6, 4, 2, 64, 32, torch.float16, 5000, False)
    q, _, tq, _ = exact(qkv, positions, inv_freq, w, 4, 2, 64, True, 1.0, torch.float16)
    d = qkv.to(gpu)
    ops.rotary(d[:, :256], None, positions.to(gpu), inv_freq.to(gpu), 4, 0, 64, interleaved=True)
    LC.check(d[:, :256], q, tq, "q")
    assert torch.equal(d[:, 256:].cpu(), qkv[:, 256:])
    ops.rotary(d[:0, :256], d[:0, 256:384], positions.to(gpu)[:0], inv_freq.to(gpu), 4, 2, 64)


@pytest.mark.parametrize("far", [2 ** 24 + 1, 2 ** 31, 2 ** 40])
def test_far_positions(gpu, far):
    """The angle is the fp64 product's: positions that fp32 cannot hold."""
    inv_freq, _ = ops.rotary_inv_freq(1e4, 128)
    positions = torch.tensor([far, far + 1, far + 2])
    x = torch.randn(3, 256, generator=torch.Generator().manual_seed(1))
    q, _, tq, _ = exact(x, positions, inv_freq, [None, None], 1, 0, 128, False, 1.0, torch.float32)
    got = x[:, :128].contiguous().to(gpu)
    ops.rotary(got, None, positions.to(gpu), inv_freq.to(gpu), 1, 0, 128)
    LC.check(got, q, tq, "far")


def test_half_layout_agrees_with_qk_norm_rope(gpu):
    """At positions whose fp32 angles are near the exact ones, the reference's form gives the same."""
    qkv, positions, _, w = inputs(52, 40, 8, 2, 128, 128, torch.float32, 64, True)
    positions = positions.clamp(0, 63)
    inv32 = ops.rope_inv_freq(1e6, 128, gpu)
    a, b = qkv.to(gpu), qkv.to(gpu)
    wd = [x.to(gpu) for x in w]
    ops.qk_norm_rope(a[:, :1024], a[:, 1024:1280], positions.to(gpu), wd[0], wd[1], inv32, 8, 2, 128)
    ops.rotary(b[:, :1024], b[:, 1024:1280], positions.to(gpu), inv32.double(), 8, 2, 128, q_w=wd[0], k_w=wd[1])
    # the reference's angle is off by half an fp32 step of at most 63
    _, _, tq, tk = exact(qkv, positions, inv32.double().cpu(), w, 8, 2, 128, False, 1.0, torch.float32)
    tol = 2 * torch.from_numpy(np.concatenate([tq, tk], 1)) + 64 * U * 2 * a[:, :1280].abs().max().item()
    assert ((a[:, :1280] - b[:, :1280]).abs().cpu() <= tol).all()


def test_captured_call(gpu):
    qkv, positions, inv_freq, _ = inputs(53, 16, 28, 4, 128, 64, torch.bfloat16, 9999, False)
    d, p, f = qkv.to(gpu), positions.to(gpu), inv_freq.to(gpu)
    kc, vc = (torch.zeros(64, 4, 128, dtype=torch.bfloat16, device=gpu) for _ in range(2))
    slots = torch.arange(16, dtype=torch.int32, device=gpu)
    qo = torch.empty(16, 28 * 128, dtype=torch.bfloat16, device=gpu)
    call = lambda: ops.rotary_store_kv(d[:, :3584], d[:, 3584:4096], d[:, 4096:], p, f, 28, 4, 128, kc, vc, slots,  # noqa: E731
                                       interleaved=True, q_out=qo)
    call()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    for step in range(3):
        p += 1
        slots += 16
        g.replay()
        torch.cuda.synchronize()
        got, at = (qo.clone(), kc.clone(), vc.clone()), None
        call()
        assert all(torch.equal(x, y) for x, y in zip(got, (qo, kc, vc)))
