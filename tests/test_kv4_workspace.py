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


@pytest.mark.parametrize("qh,kvh,hd", [(32, 8, 128), (28, 4, 128), (14, 2, 64), (8, 8, 128), (40, 2, 64)])
@pytest.mark.parametrize("tokens", [8, 160, 500, 3000])
def test_any_bound_of_the_query_lengths(tokens, qh, kvh, hd):
    """max_query_len bounds the sequences' tokens: short ones are possible under any bound, so a larger bound needs as much."""
    for bound in range(2, 9):
        assert size(tokens, qh, kvh, hd, max_query_len=bound) <= size(tokens, qh, kvh, hd, max_query_len=64), bound
    assert size(tokens, qh, kvh, hd, max_query_len=64) == size(tokens, qh, kvh, hd)


@pytest.mark.parametrize("tokens", [8, 64, 300])
@pytest.mark.parametrize("qh,kvh,bound", [(28, 4, 4), (16, 4, 8), (12, 2, 5)])
def test_groups_of_head_size_128(tokens, qh, kvh, bound):
    """Their waves without eight kv heads side by side are three on each of 1024 SIMDs, and as many hold states at once."""
    assert size(tokens, qh, kvh, 128, max_query_len=bound) <= (tokens * qh + 3 * 1024 * 16) * 130 * 4 + 16 * tokens
