"""The long-context operators together, as a serving step uses them: positions rotated and stored, a
prompt forked into samples, their shared prefix read once, pages out of the window given back, the pool
moved together, and the window read through the new tables."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("qh,kvh,hd,bs", [(14, 2, 64, 16), (28, 4, 128, 64), (6, 3, 80, 8)])
def test_serving_steps(gpu, dt, qh, kvh, hd, bs):
    g = torch.Generator().manual_seed(7)
    prompt, samples, window, sinks, pages = 150, 5, 48, 4, 80
    qn, kn, rot, scale = qh * hd, kvh * hd, hd // 2 // 2 * 2, hd ** -0.5
    inv_freq, attn = ops.rotary_inv_freq(1e6, rot, ops.ROPE_RAMP, 4.0, 1.0, 32.0, 8192.0, device=gpu)
    kc, vc = (torch.full((pages * bs, kvh, hd), float("nan"), dtype=dt, device=gpu) for _ in range(2))
    cols = -(-(prompt + 8) // bs)
    table = torch.full((samples + 1, cols), -1, dtype=torch.int32, device=gpu)
    key_len = torch.zeros(samples + 1, dtype=torch.int32, device=gpu)
    ref = torch.zeros(pages, dtype=torch.int32, device=gpu)
    first = torch.randperm(pages, generator=g)[:-(-prompt // bs)].int().to(gpu)
    table[0, :len(first)] = first
    ref[first.long()] = 1
    key_len[0] = prompt

    def tokens(n):
        return torch.randn((n, qn + 2 * kn), generator=g).to(dt).to(gpu)

    def store(qkv, seq, pos):
        slots = (table[seq.long(), pos // bs] * bs + pos % bs).int()
        ops.rotary_store_kv(qkv[:, :qn], qkv[:, qn:qn + kn], qkv[:, qn + kn:], pos, inv_freq, qh, kvh, hd, kc, vc, slots,
                            interleaved=True, attn_scale=attn)
        return qkv[:, :qn].unflatten(1, (qh, hd))

    def verify(got, q, seq, lens, w, s):
        b = LC.Batch(q, kc, vc, seq.cpu().numpy(), lens.cpu().numpy(), table.cpu().numpy().astype(np.int64), None, bs, scale)
        LC.check(got, *LC.exact_attention(b, w, s), "chain")

    # the prompt, attended in a window
    pos = torch.arange(prompt, device=gpu)
    seq = torch.zeros(prompt, dtype=torch.int32, device=gpu)
    q = store(tokens(prompt), seq, pos)
    lens = (pos + 1).int()
    verify(ops.window_attention(q, kc, vc, seq, lens, table, bs, scale, window, sinks), q, seq, lens, window, sinks)
    # samples of it
    new = ops.fork_pages([kc, vc], table, key_len, ref, [0] * samples, list(range(1, samples + 1)), bs)
    assert (new >= 0).all() == (prompt % bs > 0)
    seq = torch.arange(1, samples + 1, dtype=torch.int32, device=gpu)
    for step in range(3):
        n = key_len[1:].clone()
        need = (n % bs == 0).nonzero().view(-1).tolist()  # a new page for those whose last is full
        for i in need:
            page = int((ref == 0).nonzero()[0])
            table[i + 1, int(n[i]) // bs] = page
            ref[page] = 1
        q = store(tokens(samples), seq, n.long())
        key_len[1:] += 1
        lens = key_len[1:].clone()
        if step < 2:
            got = ops.prefix_attention(q, kc, vc, seq, lens, table, bs, scale, prompt)
            verify(got, q, seq, lens, 1 << 30, 0)
        else:
            got = ops.window_attention(q, kc, vc, seq, lens, table, bs, scale, window, sinks, max_query_len=1)
            verify(got, q, seq, lens, window, sinks)
    # the prompt's own sequence ends, the samples keep their windows, the pool is moved together
    ops.free_pages(table, key_len, ref, [0], bs)
    ops.free_pages(table, key_len, ref, list(range(1, samples + 1)), bs, window=window, sinks=sinks)
    used = ref > 0
    free_rows = (~used).repeat_interleave(bs)
    kc[free_rows], vc[free_rows] = float("nan"), float("nan")  # what was given back may hold anything
    before = ops.window_attention(q, kc, vc, seq, lens, table, bs, scale, window, sinks, max_query_len=1)
    assert torch.equal(before, got)
    moved = int(ops.compact_pages([kc, vc], table, ref, bs))
    assert moved == int(used[int(used.sum()):].sum()) and bool((ref[:int(used.sum())] > 0).all())
    after = ops.window_attention(q, kc, vc, seq, lens, table, bs, scale, window, sinks, max_query_len=1)
    assert torch.equal(after, got)
    verify(after, q, seq, lens, window, sinks)
