"""Window and prefix attention where tokens have no keys: key counts down to the least int32."""
from __future__ import annotations

import pytest

from nano_vllm_cpp_amd import ops
from tests import long_context as LC
from tests.test_gpu_prefix_attention import shared_batch
from tests.test_gpu_window_attention import forms

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("count", [-1, -2 ** 31 + 1, -2 ** 31])
def test_key_counts_below_zero(gpu, dt, count):
    """Tokens without keys among tokens that see whole chunks: zeros."""
    b = LC.make_batch(400, [300], [60], 14, 2, 64, 16, dt)
    b.key_len[[3, 40]] = count
    exact, tol = LC.exact_attention(b)
    d, meta = b.to(gpu), b.meta(gpu)
    for name, kw in forms(b):
        got = ops.window_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, 1 << 20, 0, **kw)
        assert not got[[3, 40]].any(), name
        LC.check(got, exact, tol, name)
    b, start = shared_batch(401, [20], [200], [1, 70] * 10, 14, 2, 64, 16, dt)
    b.key_len[[2, 13]] = count
    exact, tol = LC.exact_attention(b)
    d, meta = b.to(gpu), b.meta(gpu)
    for share in (True, False):
        got = ops.prefix_attention(d.q, d.k_cache, d.v_cache, *meta, b.bs, b.scale, [200], start, share=share)
        assert not got[[2, 13]].any()
        LC.check(got, exact, tol, f"share={share}")
