"""K and V appended to a 4-bit cache and read back, against the definition in 64 bits.

Codes and words are whole numbers, and the two computations differ by some 2^-50: they have to be equal.  The rotated q
and k_out have test_gpu_rotary's tolerance."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC
from tests import test_gpu_rotary as ROT

pytestmark = pytest.mark.gpu

# tokens, q_heads, kv_heads, head_dim, rotary_dim
SHAPES = [(1, 14, 2, 64, 64), (37, 28, 4, 128, 128), (300, 32, 8, 128, 64), (5, 3, 1, 256, 256), (9, 6, 3, 96, 32),
          (4, 5, 5, 32, 10), (33, 14, 2, 64, 32), (7, 2, 2, 128, 96), (3, 1, 1, 160, 2), (6, 4, 2, 128, 0),
          (21, 100, 3, 64, 16), (2, 4, 4, 256, 8), (1029, 7, 1, 64, 64)]


def exact_keys(qkv, positions, inv_freq, w, qh, kvh, hd, interleaved, scale, eps):
    """The rotated keys in 64 bits [tokens, kvh, hd]."""
    tokens, rot = qkv.shape[0], 2 * len(inv_freq)
    x = qkv[:, qh * hd:(qh + kvh) * hd].double().numpy().reshape(tokens, kvh, hd).copy()
    if w[1] is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w[1].double().numpy()
    angle = positions.double().numpy()[:, None] * inv_freq.numpy()
    cos, sin = (np.cos(angle) * scale)[:, None], (np.sin(angle) * scale)[:, None]
    ia, ib = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else \
        (np.arange(rot // 2), np.arange(rot // 2) + rot // 2)
    a, b = x[..., ia], x[..., ib]
    y = x.copy()
    y[..., ia], y[..., ib] = a * cos - b * sin, b * cos + a * sin
    return y


def store(gpu, qkv, positions, inv_freq, w, qh, kvh, hd, kc, vc, slots, **kw):
    """(q_out, k cache, v cache) on the host."""
    d = qkv.to(gpu)
    qn, kn = qh * hd, kvh * hd
    k, v = torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu)
    wd = [x.to(gpu) if x is not None else None for x in w]
    q_out = kw.pop("q_out", None)
    q_out = torch.empty((len(d), qn), dtype=d.dtype, device=gpu) if q_out is None else q_out
    ops.rotary_store_kv4(d[:, :qn], d[:, qn:qn + kn], d[:, qn + kn:], positions.to(gpu), inv_freq.to(gpu), qh, kvh, hd, k, v,
                         torch.from_numpy(slots).to(gpu), q_w=wd[0], k_w=wd[1], q_out=q_out, **kw)
    assert torch.equal(d.cpu().view(torch.int16 if d.element_size() == 2 else torch.int32),
                       qkv.view(torch.int16 if d.element_size() == 2 else torch.int32))  # the inputs stay
    return q_out, k.cpu().numpy(), v.cpu().numpy()


def slots_of(r, tokens):
    """Rows of a cache of tokens + 9, some tokens without one."""
    slots = r.permutation(tokens + 9)[:tokens].astype(np.int32)
    slots[2::5] = -1
    if tokens > 3:
        slots[3] = tokens + 9  # past the cache
    return slots


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("norm", [False, True], ids=["plain", "norm"])
@pytest.mark.parametrize("ci", range(len(SHAPES)))
def test_store(gpu, dt, interleaved, norm, ci):
    tokens, qh, kvh, hd, rot = SHAPES[ci]
    print(f"[case] {SHAPES[ci]}", flush=True)
    qkv, positions, inv_freq, w = ROT.inputs(ci, tokens, qh, kvh, hd, rot, dt, 1_000_000, norm)
    scale = 1.2718 if ci % 2 else 1.0
    r = np.random.default_rng(ci)
    row = kv4.row_bytes(kvh, hd)
    kc, vc = (r.integers(0, 256, (tokens + 9, row)).astype(np.uint8) for _ in range(2))
    slots = slots_of(r, tokens)
    q, k, tq, tk = ROT.exact(qkv, positions, inv_freq, w, qh, kvh, hd, interleaved, scale, dt)
    keys = exact_keys(qkv, positions, inv_freq, w, qh, kvh, hd, interleaved, scale, 1e-6)
    vals = qkv[:, (qh + kvh) * hd:].double().numpy().reshape(tokens, kvh, hd)
    want_k, want_v = kc.copy(), vc.copy()
    kept = (slots >= 0) & (slots < tokens + 9)
    want_k[slots[kept]] = kv4.pack(*kv4.quantize(keys))[kept]
    want_v[slots[kept]] = kv4.pack(*kv4.quantize(vals))[kept]
    k_out = torch.empty((tokens, kvh * hd), dtype=dt, device=gpu) if ci % 3 else None
    got_q, got_k, got_v = store(gpu, qkv, positions, inv_freq, w, qh, kvh, hd, kc, vc, slots, interleaved=interleaved,
                                attn_scale=scale, k_out=k_out)
    LC.check(got_q, q, tq, "q_out")
    if k_out is not None:
        LC.check(k_out, k, tk, "k_out")
    used = kvh * (hd // 2 + hd // 16)  # (a row's padding may change)
    for name, got, want in (("v", got_v, want_v), ("k", got_k, want_k)):
        bad = np.argwhere(got[:, :used] != want[:, :used])
        assert len(bad) == 0, f"{name}: {len(bad)} bytes differ, first {bad[0]}"
    # what the rows stand for
    for dtype in LC.DTYPES:
        back = ops.kv4_unpack(torch.from_numpy(got_v).to(gpu), kvh, hd, dtype)
        exact = kv4.values(got_v, kvh, hd)
        want = torch.from_numpy(np.nan_to_num(exact, nan=0.0, posinf=0.0, neginf=0.0)).to(dtype)
        fine = torch.from_numpy(np.isfinite(exact))
        assert torch.equal(torch.where(fine, back.cpu(), torch.zeros((), dtype=dtype))[slots[kept]], want[slots[kept]])


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("hd", [64, 128, 96, 256])
def test_extreme_values(gpu, dt, hd):
    """Zeros, ties, one sign, tiny and huge spans, infinities and NaN in one group, and no rotation."""
    kvh, groups = 2, 2 * hd // 32
    r = np.random.default_rng(hd)
    rows = []
    for scale in (0.0, 1e-9, 2.0 ** -24, 2.0 ** -16, 6e-5, 1e-3, 0.3, 1.0, 17.0, 900.0, 4000.0, 30000.0, 65000.0):
        for kind in range(4):
            x = r.standard_normal((groups, 32)) * scale
            if kind == 1:
                x = np.abs(x)
            if kind == 2:
                x = -np.abs(x)
            if kind == 3:  # ties: halves of a step
                x = np.rint(np.clip(x, -65000, 65000) * 4) / 4
            rows.append(x.reshape(kvh, hd))
    x = np.stack(rows)
    bad = x[:3].copy()
    bad[0, 0, 5], bad[1, 1, hd - 1], bad[2, 0, 31], bad[2, 0, 32] = np.inf, np.nan, -np.inf, 1e4
    x = np.concatenate([x, bad])
    t = torch.from_numpy(np.clip(x, -65504, 65504) if dt == torch.float16 else x).to(dt)
    t[-3:] = torch.from_numpy(bad).to(dt)
    tokens = len(t)
    flat = t.reshape(tokens, -1).to(gpu)
    kc, vc = ops.kv4_cache(tokens, kvh, hd, gpu), ops.kv4_cache(tokens, kvh, hd, gpu)
    slots = torch.arange(tokens, dtype=torch.int32, device=gpu)
    ops.rotary_store_kv4(flat.clone(), flat, flat, torch.zeros(tokens, dtype=torch.int64, device=gpu),
                         torch.zeros(0, dtype=torch.float64, device=gpu), kvh, kvh, hd, kc, vc, slots)
    want = kv4.pack(*kv4.quantize(t.double().numpy()))
    for name, c in (("v", vc), ("k", kc)):
        got = c.cpu().numpy()
        bad = np.argwhere(got != want)
        assert len(bad) == 0, f"{name}: {len(bad)} bytes differ, first {bad[0]}"
    # within half a step of the value where the scale reaches
    back = kv4.values(want, kvh, hd)[:-3]
    v = t.double().numpy()[:-3].reshape(-1, 32)
    spread = np.maximum(v.max(-1), 0) - np.minimum(v.min(-1), 0)
    fits = spread / 15 <= 4352
    step = spread / 15 + np.maximum(spread / 15 * 2.0 ** -6, 2.0 ** -20)
    assert (np.abs(back.reshape(-1, 32) - v)[fits] <= 0.5001 * step[fits, None]).all()


def test_in_place_strided_and_empty(gpu):
    """q and k rotated in place in packed rows with a gap, on another stream; no tokens."""
    tokens, qh, kvh, hd, dt = 50, 6, 2, 64, torch.bfloat16
    qkv, positions, inv_freq, w = ROT.inputs(3, tokens, qh, kvh, hd, hd, dt, 5000, True)
    width = (qh + 2 * kvh) * hd
    wide = torch.randn((tokens, width + 24)).to(dt)
    wide[:, 8:8 + width] = qkv
    q, k, tq, tk = ROT.exact(qkv, positions, inv_freq, w, qh, kvh, hd, False, 1.0, dt)
    qn, kn = qh * hd, kvh * hd
    for offset in (8, 3):  # 16-byte rows, and odd ones
        d = torch.empty((tokens, width + 24), dtype=dt, device=gpu)
        d[:, offset:offset + width] = qkv.to(gpu)
        s = d[:, offset:offset + width]
        kc, vc = ops.kv4_cache(tokens, kvh, hd, gpu), ops.kv4_cache(tokens, kvh, hd, gpu)
        slots = torch.arange(tokens, dtype=torch.int32, device=gpu).flip(0).contiguous()
        args = (positions.to(gpu), inv_freq.to(gpu), qh, kvh, hd, kc, vc, slots)
        weights = dict(q_w=w[0].to(gpu), k_w=w[1].to(gpu))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            ops.rotary_store_kv4(s[:, :qn], s[:, qn:qn + kn], s[:, qn + kn:], *args, k_out=s[:, qn:qn + kn], **weights)
        stream.synchronize()
        LC.check(s[:, :qn], q, tq, "q in place")
        LC.check(s[:, qn:qn + kn], k, tk, "k in place")
        assert torch.equal(s[:, qn + kn:].cpu(), qkv[:, qn + kn:])
        keys = exact_keys(qkv, positions, inv_freq, w, qh, kvh, hd, False, 1.0, 1e-6)
        assert np.array_equal(kc.cpu().numpy()[::-1], kv4.pack(*kv4.quantize(keys)))
        ops.rotary_store_kv4(s[:0, :qn], s[:0, qn:qn + kn], s[:0, qn + kn:], args[0][:0], *args[1:7], slots[:0], **weights)
        assert ops.kv4_unpack(kc[:0], kvh, hd).shape == (0, kvh, hd)
