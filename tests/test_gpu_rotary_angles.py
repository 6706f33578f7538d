"""The sine and cosine of rotary positions, to fp32's precision at every angle.

With a pair (1, 0) and scale 1 the outputs are the cosine and the sine.  Tolerance, with u = 2^-24: the fp32 functions'
documented 2 units (4 u of the value), the correction by what rounding the reduced angle left, its sum and the
scale (2 u), 2^-51 |angle| from the fp64 product and reduction, and 4 u of the reduced angle r's own rounding (at most
2^-23), by which the functions' values differ from the result: 2^-45.  Nothing of the order of that rounding itself,
which near a zero is many units of the value."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("hd", [128, 96])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
def test_sine_and_cosine(gpu, hd, interleaved):
    inv_freq, _ = ops.rotary_inv_freq(1e4, hd)
    g = torch.Generator().manual_seed(3)
    positions = torch.cat([torch.arange(600), torch.randint(0, 1_000_000, (600,), generator=g)])
    x = torch.zeros(len(positions), hd)
    ia, ib = (np.arange(0, hd, 2), np.arange(1, hd, 2)) if interleaved else (np.arange(hd // 2), np.arange(hd // 2) + hd // 2)
    x[:, ia] = 1.0
    got = x.to(gpu)
    ops.rotary(got, None, positions.to(gpu), inv_freq.to(gpu), 1, 0, hd, interleaved=interleaved)
    y = got.double().cpu().numpy()
    angle = positions.double().numpy()[:, None] * inv_freq.numpy()
    for name, have, want in (("cos", y[:, ia], np.cos(angle)), ("sin", y[:, ib], np.sin(angle))):
        off = np.abs(have - want)
        tol = 6 * U * np.abs(want) + 2.0 ** -51 * np.abs(angle) + 2.0 ** -45
        assert (off <= tol).all(), (name, float((off / tol).max()))
