"""Shared by the tests of the window and prefix attention, the cache pages and the rotary positions:
paged batches whose unseen cache rows are poisoned, and the operators' definitions in 64 bits."""
from __future__ import annotations

import dataclasses

import numpy as np
import torch

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
DT_IDS = ["f32", "f16", "bf16"]


def half_step(dt: torch.dtype) -> float:
    """The most that a value is off, relative to itself, after one rounding to dt."""
    return torch.finfo(dt).eps / 2


@dataclasses.dataclass
class Batch:
    q: torch.Tensor            # [tokens, q_heads, hd]
    k_cache: torch.Tensor      # [blocks * bs, kv_heads, hd]
    v_cache: torch.Tensor
    seq: np.ndarray            # [tokens]
    key_len: np.ndarray        # [tokens]
    table: np.ndarray          # [seqs, max_blocks]
    cu: np.ndarray             # [seqs + 1]
    bs: int
    scale: float

    def to(self, device):
        return dataclasses.replace(self, q=self.q.to(device), k_cache=self.k_cache.to(device),
                                   v_cache=self.v_cache.to(device))

    def meta(self, device):
        return [torch.from_numpy(np.ascontiguousarray(x.astype(np.int32))).to(device)
                for x in (self.seq, self.key_len, self.table)]


def seen_keys(n: int, window: int, sinks: int) -> np.ndarray:
    """Truth values over the keys of a token with n keys."""
    j = np.arange(max(n, 0))
    return (j >= n - window) | (j < sinks)


def make_batch(seed, ctx, new, q_heads, kv_heads, hd, bs, dt, window=1 << 30, sinks=0, extra=3, key_len=None,
               std=1.0) -> Batch:
    """Sequences of ctx[s] keys, the last new[s] of them queried.  Every cache row that holds no key seen by
    a token of the batch is NaN, and the table entries of pages without such a key are no pages."""
    g = torch.Generator().manual_seed(seed)
    r = np.random.default_rng(seed)
    ctx, new = np.asarray(ctx), np.asarray(new)
    seq = np.repeat(np.arange(len(ctx)), new)
    if key_len is None:
        key_len = np.concatenate([np.arange(c - n, c) + 1 for c, n in zip(ctx, new)] or [np.zeros(0)]).astype(np.int64)
    blocks = -(-ctx // bs)
    table = r.choice([-1, -7, 1 << 30], (len(ctx), max(1, int(blocks.max(initial=0))) + 1)).astype(np.int64)
    rows = int(blocks.sum() + extra) * bs
    k = torch.full((rows, kv_heads, hd), float("nan"))
    v = torch.full((rows, kv_heads, hd), float("nan"))
    free = list(r.permutation(int(blocks.sum()) + extra))
    for s, c in enumerate(ctx):
        some = np.zeros(int(c), bool)
        for n in key_len[seq == s]:
            some[:max(n, 0)] |= seen_keys(int(n), window, sinks)
        for b in range(int(blocks[s])):
            js = np.flatnonzero(some[b * bs:(b + 1) * bs])
            if len(js):
                page = free.pop()
                table[s, b] = page
                at = torch.from_numpy(page * bs + js)
                k[at] = torch.randn((len(js), kv_heads, hd), generator=g) * std
                v[at] = torch.randn((len(js), kv_heads, hd), generator=g)
    q = torch.randn((len(seq), q_heads, hd), generator=g) * std
    return Batch(q.to(dt), k.to(dt), v.to(dt), seq, np.asarray(key_len), table,
                 np.concatenate([[0], np.cumsum(new)]).astype(np.int32), bs, hd ** -0.5)


def exact_attention(b: Batch, window: int = 1 << 30, sinks: int = 0):
    """(out, tolerance) in 64 bits.

    The tolerance, for fp32 sums and P rounded once to the storage type t before P . V:
      scores: (hd + 8) roundings of 2^-24 of S = scale max sum |q k| move each exponent, and p by as much
              relatively; twice that on out, relative to max |V|;
      sums:   n + 8 roundings of 2^-24 of sum p |V| / sum p <= max |V|;
      P:      half a step of t relatively (fp16 also 2^-25 absolutely below 2^-14, n of them);
      out:    half a step of t of its own value (and the least subnormal's half)."""
    dt = b.q.dtype
    tokens, q_heads, hd = b.q.shape
    kv_heads = b.k_cache.shape[1]
    group = q_heads // kv_heads
    out, tol = np.zeros(b.q.shape), np.zeros(b.q.shape)
    q, kc, vc = (x.double().cpu().numpy() for x in (b.q, b.k_cache, b.v_cache))
    for t in range(tokens):
        n = int(b.key_len[t])
        j = np.flatnonzero(seen_keys(n, window, sinks))
        if not len(j):
            continue
        rows = b.table[b.seq[t], j // b.bs] * b.bs + j % b.bs
        for h in range(kv_heads):
            qh, k, v = q[t, h * group:(h + 1) * group], kc[rows, h], vc[rows, h]
            s = qh @ k.T * b.scale
            p = np.exp(s - s.max(1, keepdims=True))
            o = p @ v / p.sum(1, keepdims=True)
            out[t, h * group:(h + 1) * group] = o
            S = b.scale * (np.abs(qh) @ np.abs(k).T).max()
            e = 2 * (hd + 8) * 2.0 ** -24 * S + (len(j) + 8) * 2.0 ** -24
            if dt != torch.float32:
                e += half_step(dt)
            if dt == torch.float16:
                e += len(j) * 2.0 ** -25
            tiny = 2.0 ** -25 if dt == torch.float16 else 1e-30
            tol[t, h * group:(h + 1) * group] = e * np.abs(v).max() + half_step(dt) * np.abs(o) + tiny
    return out, tol


def check(got: torch.Tensor, exact: np.ndarray, tol: np.ndarray, what: str) -> None:
    g = got.double().cpu().numpy()
    bad = ~(np.abs(g - exact) <= tol)
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {bad.size} outside the tolerance; first {i}: got {g[i]!r}, exact "
                             f"{exact[i]!r}, tolerance {tol[i]!r}")
