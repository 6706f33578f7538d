"""Prefix attention's launches: tiles and tokens in one, and calls of more workgroups than go into one."""
from __future__ import annotations

import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import long_context as LC
from tests.test_gpu_prefix_attention import shared_batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
def test_prefix_calls_of_many_workgroups(gpu, dt):
    """65600 tokens of 32 kv heads over one sequence: more than 2^21 workgroups, so tiles and tokens in launches of
    their own."""
    tokens, heads, hd, bs, prefix, most = 65600, 32, 64, 16, 40, 64
    g = torch.Generator(device=gpu).manual_seed(7)
    q = torch.randn((tokens, heads, hd), generator=g, device=gpu).to(dt)
    k, v = (torch.randn((6 * bs, heads, hd), generator=g, device=gpu).to(dt) for _ in range(2))
    table = torch.tensor([[4, 1, 5, 2]], dtype=torch.int32, device=gpu)
    seq = torch.zeros(tokens, dtype=torch.int32, device=gpu)
    n = torch.randint(0, most + 1, (tokens,), generator=g, device=gpu, dtype=torch.int32)
    assert tokens * heads > 1 << 21
    got = ops.prefix_attention(q, k, v, seq, n, table, bs, hd ** -0.5, prefix)
    at = (table[0].long()[:, None] * bs + torch.arange(bs, device=gpu)).view(-1)
    seen = torch.arange(most, device=gpu) < n[:, None]
    some = n > 0
    assert not got[~some].any()
    step = LC.half_step(dt)
    for h in range(heads):  # the bound is long_context.exact_attention's
        qh, kh, vh = q[:, h].double(), k[at, h].double(), v[at, h].double()
        s = torch.where(seen, qh @ kh.T.contiguous() * hd ** -0.5, -torch.inf)[some]
        o = torch.softmax(s, 1) @ vh
        S = hd ** -0.5 * (qh[some].abs() @ kh.T.contiguous().abs()).amax(1, keepdim=True)
        e = 2 * (hd + 8) * 2.0 ** -24 * S + (most + 8) * 2.0 ** -24 + step + most * 2.0 ** -25
        tol = e * vh.abs().max() + step * o.abs() + 2.0 ** -25
        assert ((got[some, h].double() - o).abs() <= tol).all(), h


@pytest.mark.parametrize("hd", [64, 128])
def test_fp32_calls_of_some_workgroups(gpu, hd):
    """Over 256 workgroups: at head size 64 tiles and tokens share a launch, at 128 they do not."""
    b, start = shared_batch(500, [70, 1, 30], [500, 64, 129], [1, 130, 40, 300] * 25 + [9], 14, 2, hd, 16, torch.float32)
    exact, tol = LC.exact_attention(b)
    d, meta = b.to(gpu), b.meta(gpu)
    for share in (True, False):
        got = ops.prefix_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, [500, 64, 129], start, share=share)
        LC.check(got, exact, tol, f"share={share}")
