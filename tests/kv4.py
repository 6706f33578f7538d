"""The 4-bit cache's rows and the attention over them from their definitions in 64 bits (numpy), for the tests."""
from __future__ import annotations

import numpy as np
import torch

from tests import long_context as LC

GROUP = 32
NOT_A_NUMBER = 0x7E00


def row_bytes(kvh: int, hd: int) -> int:
    return (kvh * hd // 2 + kvh * (hd // GROUP) * 2 + 15) // 16 * 16


def scale_bits(d: np.ndarray) -> np.ndarray:
    return d.astype(np.float16).view(np.uint16).astype(np.int64)


def quantize(x: np.ndarray):
    """(codes [rows, kvh, hd], words [rows, kvh, hd / 32]) of values [rows, kvh, hd]."""
    rows, kvh, hd = x.shape
    x = x.astype(np.float64).reshape(rows, kvh, hd // GROUP, GROUP)
    fine = np.isfinite(x).all(-1)
    x = np.where(fine[..., None], x, 0.0)
    low, high = np.minimum(x.min(-1), 0.0), np.maximum(x.max(-1), 0.0)
    need = (high - low) / 15.0
    _, expo = np.frexp(need)  # need in [2^(expo - 1), 2^expo): seven bits are multiples of 2^(expo - 7)
    step = np.ldexp(1.0, np.maximum(expo - 7, -20))
    d = np.minimum(np.ceil(need / step) * step, 4352.0)
    one = np.where(d > 0, d, 1.0)
    z = np.minimum(np.rint(-low / one), 15.0)
    n = np.clip(np.rint(x / one[..., None]) + z[..., None], 0, 15)
    words = np.where(fine, scale_bits(d) | z.astype(np.int64), NOT_A_NUMBER)
    return np.where(fine[..., None], n, 0).astype(np.int64).reshape(rows, kvh, hd), words


def pack(codes: np.ndarray, words: np.ndarray) -> np.ndarray:
    rows, kvh, hd = codes.shape
    out = np.zeros((rows, row_bytes(kvh, hd)), np.uint8)
    n = codes.reshape(rows, kvh * hd)
    out[:, :kvh * hd // 2] = n[:, 0::2] | n[:, 1::2] << 4
    w = words.reshape(rows, -1)
    at = kvh * hd // 2
    out[:, at:at + 2 * w.shape[1]:2], out[:, at + 1:at + 2 * w.shape[1]:2] = w & 255, w >> 8
    return out


def values(cache: np.ndarray, kvh: int, hd: int) -> np.ndarray:
    """[rows, kvh, hd] in 64 bits."""
    rows = len(cache)
    codes = cache[:, :kvh * hd // 2].astype(np.int64)
    n = np.stack([codes & 15, codes >> 4], -1).reshape(rows, kvh, hd // GROUP, GROUP)
    at, words = kvh * hd // 2, kvh * (hd // GROUP)
    w = cache[:, at:at + 2 * words].astype(np.uint16)
    w = (w[:, 0::2] | w[:, 1::2] << 8).reshape(rows, kvh, hd // GROUP)
    d = (w & 0xFFF0).astype(np.uint16).view(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return (d[..., None] * (n - (w & 15).astype(np.int64)[..., None])).reshape(rows, kvh, hd)


def poisoned(x: torch.Tensor, r: np.random.Generator) -> np.ndarray:
    """The 4-bit rows of x [rows, kvh, hd]; rows that hold a NaN get any bytes, most scales no numbers."""
    v = x.double().numpy()
    out = pack(*quantize(v))
    rows, kvh, hd = v.shape
    bad = np.isnan(v).any((1, 2))
    junk = r.integers(0, 256, (int(bad.sum()), out.shape[1])).astype(np.uint8)
    at, words = kvh * hd // 2, kvh * (hd // GROUP)
    high = r.choice([0x7C, 0x7E, 0xFC, 0xFF, 0x7F, 0x3A], (len(junk), words))
    junk[:, at + 1:at + 2 * words:2] = high
    out[bad] = junk
    return out


def make_batch(seed, ctx, new, qh, kvh, hd, bs, dt, key_len=None, std=1.0):
    """(long_context.Batch with the caches' values in 64 bits, K rows, V rows): unseen rows hold anything."""
    b = LC.make_batch(seed, ctx, new, qh, kvh, hd, bs, torch.float32, key_len=key_len, std=std)
    r = np.random.default_rng(seed)
    kc, vc = poisoned(b.k_cache, r), poisoned(b.v_cache, r)
    b.q = b.q.to(dt)
    b.k_cache, b.v_cache = torch.from_numpy(values(kc, kvh, hd)), torch.from_numpy(values(vc, kvh, hd))
    return b, kc, vc


def exact_attention(b: LC.Batch, one_part: bool):
    """(out, tolerance) in 64 bits of paged attention over values b.k_cache, b.v_cache.

    The tolerance, u = 2^-24:
      q:      exact in fp16 after its scaling by a power of two, but for 2^-24 absolutely where its row's largest is at least
              2^10: 2^-34 of the largest; fp32 as two fp16 numbers, 2^-22 relatively as well;
      scores: (hd + 8) u of S = scale max sum |q k| in all, and q's part; they move each exponent, so p by as much
              relatively, and out by twice that relative to max |V|;
      sums:   n + 8 roundings u of sum p |V| / sum p <= max |V|;
      P:      2^-22 relatively and 2^-25 absolutely (n of them, the sum of weights at least 1); 2^-11 relatively where `one_part`;
      out:    half a step of the type of its own value (and the least subnormal's half)."""
    dt = b.q.dtype
    tokens, q_heads, hd = b.q.shape
    kv_heads = b.k_cache.shape[1]
    group = q_heads // kv_heads
    out, tol = np.zeros(b.q.shape), np.zeros(b.q.shape)
    q, kc, vc = (x.double().cpu().numpy() for x in (b.q, b.k_cache, b.v_cache))
    u = 2.0 ** -24
    for t in range(tokens):
        n = int(b.key_len[t])
        if n <= 0:
            continue
        j = np.arange(n)
        rows = b.table[b.seq[t], j // b.bs] * b.bs + j % b.bs
        for h in range(kv_heads):
            qh, k, v = q[t, h * group:(h + 1) * group], kc[rows, h], vc[rows, h]
            s = qh @ k.T * b.scale
            p = np.exp(s - s.max(1, keepdims=True))
            o = p @ v / p.sum(1, keepdims=True)
            out[t, h * group:(h + 1) * group] = o
            S = abs(b.scale) * (np.abs(qh) @ np.abs(k).T).max()
            e_q = 2.0 ** -34 * abs(b.scale) * hd * np.abs(qh).max() * np.abs(k).max()
            if dt == torch.float32:
                e_q += 2.0 ** -22 * S
            e = 2 * ((hd + 8) * u * S + e_q) + (n + 8) * u + n * 2.0 ** -25 + (2.0 ** -11 if one_part else 2.0 ** -22)
            tiny = 2.0 ** -25 if dt == torch.float16 else 1e-30
            tol[t, h * group:(h + 1) * group] = e * np.abs(v).max() + LC.half_step(dt) * np.abs(o) + tiny
    return out, tol
