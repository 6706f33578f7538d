"""4-bit attention over queries and scales at the ends of their types."""
from __future__ import annotations

import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC

pytestmark = pytest.mark.gpu

FORMS = [([75, 33], [1, 1]), ([75, 33], [3, 2]), ([75, 60], [40, 9])]


def on(gpu, b, kc, vc, **kw):
    return ops.paged_attention_kv4(b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), b.k_cache.shape[1],
                                   *b.meta(gpu), b.bs, b.scale, **kw)


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("hd", [64, 128, 96])
@pytest.mark.parametrize("ctx,new", FORMS, ids=["single", "few", "chunk"])
def test_scores_that_vanish(gpu, dt, hd, ctx, new):
    """The smallest queries times the smallest scales: equal weights, and masked keys stay masked."""
    b, kc, vc = kv4.make_batch(1, ctx, new, 8, 2, hd, 16, dt)
    b.q = (torch.sign(b.q.float()) * (2.0 ** -24 if dt == torch.float16 else 2.0 ** -125)).to(dt)
    for b.scale in (2.0 ** -20, 2.0 ** -120):
        for kw in (dict(cu_seqlens=b.cu), {}):
            LC.check(on(gpu, b, kc, vc, **kw), *kv4.exact_attention(b, dt != torch.float32 and len(b.q) > 2), str(kw))


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ctx,new", FORMS, ids=["single", "few", "chunk"])
def test_zero_scores_of_large_queries(gpu, dt, ctx, new):
    """Keys of zeros: their scores are zero whatever the query and the scale."""
    b, kc, vc = kv4.make_batch(2, ctx, new, 8, 2, 128, 16, dt)
    kc[:] = 0
    b.k_cache.zero_()
    b.q = (torch.sign(b.q.float()) * (2.0 ** 15 if dt == torch.float16 else 2.0 ** 126)).to(dt)
    for b.scale in (2.0 ** 20, 2.0 ** 120):
        LC.check(on(gpu, b, kc, vc, cu_seqlens=b.cu), *kv4.exact_attention(b, dt != torch.float32 and len(b.q) > 2), "zeros")
