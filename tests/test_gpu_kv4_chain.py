"""A serving step with a 4-bit cache: prompts appended and attended over their own rows, then chunks and single tokens over
the cache, a fork with its partial page copied, pages given back and moved together."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC
from tests import test_gpu_prompt_attention as PROMPT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("qh,kvh,hd,bs", [(14, 2, 64, 16), (28, 4, 128, 64), (6, 3, 96, 8)])
def test_serving_steps(gpu, dt, qh, kvh, hd, bs):
    g = torch.Generator().manual_seed(3)
    lens, pages, cols, scale = [70, 33], 60, 24, hd ** -0.5
    qn, kn = qh * hd, kvh * hd
    inv_freq, attn = ops.rotary_inv_freq(1e6, hd, ops.ROPE_RAMP, 4.0, 1.0, 32.0, 8192.0, device=gpu)
    kc, vc = ops.kv4_cache(pages * bs, kvh, hd, gpu), ops.kv4_cache(pages * bs, kvh, hd, gpu)
    table = torch.full((4, cols), -1, dtype=torch.int32, device=gpu)
    key_len = torch.zeros(4, dtype=torch.int32, device=gpu)
    ref = torch.zeros(pages, dtype=torch.int32, device=gpu)

    def grow(seq, n):
        """Pages for n keys of the sequence, the highest free ones (so that there is something to move)."""
        for b in range(-(-n // bs)):
            if int(table[seq, b]) < 0:
                page = int((ref == 0).nonzero()[-1])
                table[seq, b] = page
                ref[page] = 1

    def append(seq, pos):
        """New tokens of the sequences, rotated and stored: (q, rotated k, v)."""
        qkv = torch.randn((len(seq), qn + 2 * kn), generator=g).to(dt).to(gpu)
        for s, p in zip(seq.tolist(), pos.tolist()):
            grow(s, p + 1)
        slots = (table[seq.long(), pos // bs] * bs + pos % bs).int()
        q, k, v = qkv[:, :qn], qkv[:, qn:qn + kn], qkv[:, qn + kn:]
        ops.rotary_store_kv4(q, k, v, pos, inv_freq, qh, kvh, hd, kc, vc, slots, attn_scale=attn, k_out=k)
        # the cache holds what the rotated rows give: v exactly as defined; k within a step of the rounded k
        rows = slots.long()
        assert np.array_equal(vc[rows].cpu().numpy(), kv4.pack(*kv4.quantize(v.double().cpu().numpy().reshape(-1, kvh, hd))))
        for s in set(seq.tolist()):
            key_len[s] = int(pos[seq == s].max()) + 1
        return q.unflatten(1, (qh, hd)), k.unflatten(1, (kvh, hd)), v.unflatten(1, (kvh, hd))

    def attend(q, seq, lens, **kw):
        got = ops.paged_attention_kv4(q, kc, vc, kvh, seq, lens, table, bs, scale, **kw)
        one = dt != torch.float32 and kw.get("max_query_len") != 1 and len(q) * (qh // kvh) > 16
        b = LC.Batch(q, *(torch.from_numpy(kv4.values(c.cpu().numpy(), kvh, hd)) for c in (kc, vc)), seq.cpu().numpy(),
                     lens.cpu().numpy(), table.cpu().numpy().astype(np.int64), None, bs, scale)
        LC.check(got, *kv4.exact_attention(b, one), "chain")
        return got

    # the prompts: stored in 4 bits, attended over their own rows
    cu = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    seq = torch.from_numpy(np.repeat([0, 1], lens).astype(np.int32)).to(gpu)
    pos = torch.from_numpy(np.concatenate([np.arange(n) for n in lens])).to(gpu)
    q, k, v = append(seq, pos)
    got = ops.prompt_attention(q, k, v, torch.from_numpy(cu).to(gpu), scale)
    LC.check(got, *PROMPT.exact(q.cpu(), k.cpu(), v.cpu(), cu.tolist(), scale), "prompts")
    # a chunk of the first sequence over the cache
    n = 21
    seq = torch.zeros(n, dtype=torch.int32, device=gpu)
    pos = torch.arange(lens[0], lens[0] + n, device=gpu)
    q, _, _ = append(seq, pos)
    attend(q, seq, (pos + 1).int())
    # the second one forked twice, and single tokens of all
    new = ops.fork_pages([kc, vc], table, key_len, ref, [1, 1], [2, 3], bs)
    assert (new >= 0).all()
    seq = torch.arange(4, dtype=torch.int32, device=gpu)
    for step in range(3):
        if step == 2:  # pages of a sequence that ended are given back, the others move together
            ops.free_pages(table, key_len, ref, [1], bs)
            before = attend(q, seq[1:], key_len[1:].clone() * (seq[1:] != 1), max_query_len=1)
            assert int(ops.compact_pages([kc, vc], table, ref, bs)) > 0
            after = attend(q, seq[1:], key_len[1:].clone() * (seq[1:] != 1), max_query_len=1)
            assert torch.equal(before, after)
            break
        q, _, _ = append(seq, key_len.long())
        attend(q, seq, key_len.clone(), max_query_len=1)
        q = q[1:].clone()
