"""Workspaces of the 4-bit attention (host only)."""
from __future__ import annotations

import pytest

from nano_vllm_cpp_amd import ops


def size(tokens, qh, kvh, hd, bs=64, max_blocks=512, max_query_len=0):
    return ops.lib().nvf_paged_attention_kv4_workspace_size(tokens, qh, kvh, hd, bs, max_blocks, max_query_len)


@pytest.mark.parametrize("qh,kvh,hd", [(16, 8, 256), (4, 4, 256), (32, 4, 256), (8, 1, 256), (14, 2, 256)])
@pytest.mark.parametrize("tokens", [2, 100, 700, 2048])
def test_states_that_can_be_written(tokens, qh, kvh, hd):
    """Tokens that share out their keys need a state for each (token, head), and one for each of 16 columns of the GPU's 4096
    waves, each of which begins one group of tokens that another wave has too."""
    assert size(tokens, qh, kvh, hd) <= (tokens * qh + 4096 * 16) * (hd + 2) * 4
