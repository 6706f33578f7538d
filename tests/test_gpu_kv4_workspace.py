"""4-bit attention with workspaces of all sizes: as large as asked for, smaller, none; nothing behind them is written."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4
from tests import long_context as LC

pytestmark = pytest.mark.gpu

# ctx, new, q_heads, kv_heads, head_dim, max_query_len
CASES = [
    ([900, 33, 400, 7], [1] * 4, 28, 4, 128, 1),
    ([900, 60, 400, 17], [5] * 4, 32, 8, 128, 64),
    ([900, 60, 400, 17], [5, 2, 3, 1], 14, 2, 64, 0),
    ([700, 90], [40, 5], 8, 4, 256, 0),
    ([900, 300], [50, 30], 14, 2, 64, 64),
]


@pytest.mark.parametrize("dt", LC.DTYPES, ids=LC.DT_IDS)
@pytest.mark.parametrize("ci", range(len(CASES)))
def test_workspaces(gpu, dt, ci):
    ctx, new, qh, kvh, hd, bound = CASES[ci]
    b, kc, vc = kv4.make_batch(ci, ctx, new, qh, kvh, hd, 16, dt)
    out, tol = kv4.exact_attention(b, dt != torch.float32 and bound != 1)
    q, k, v, meta = b.q.to(gpu), torch.from_numpy(kc).to(gpu), torch.from_numpy(vc).to(gpu), b.meta(gpu)
    tokens = len(b.q)
    full = ops.lib().nvf_paged_attention_kv4_workspace_size(tokens, qh, kvh, hd, 16, b.table.shape[1], bound)
    assert full > 0
    ws = torch.empty(full // 4 + 1024, dtype=torch.int32, device=gpu)
    stream = torch.cuda.current_stream().cuda_stream
    for cu in (b.cu, None):
        for size in sorted({full, full * 3 // 4, full // 2, full // 4, full // 16, 4 * tokens * qh * (hd + 2), 400, 0}):
            print(f"[case] {ci}: {size} of {full} bytes, packing {cu is not None}", flush=True)
            ws.fill_(-77)
            got = torch.empty_like(q)
            rc = ops.lib().nvf_paged_attention_kv4_ws(
                q.data_ptr(), got.data_ptr(), k.data_ptr(), v.data_ptr(), *(m.data_ptr() for m in meta),
                cu.ctypes.data if cu is not None else None, len(ctx), tokens, qh, kvh, hd, 16, b.table.shape[1],
                len(kc) // 16, b.scale, q.stride(0), bound, ws.data_ptr(), size, ops._dt(q), stream)
            assert rc == 0
            LC.check(got, out, tol, f"{size} of {full} bytes")
            assert (ws[-(-size // 4):] == -77).all(), f"{size} of {full} bytes"
