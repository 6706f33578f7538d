"""Refusals of the long-context operators (host only: no call here reaches a launch) and the frequency
tables of scaled rotary positions."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops

P = 0x1000  # never dereferenced


def refused(rc, text):
    msg = ops.lib().nvf_last_error().decode()
    assert rc == -1 and text in msg, (rc, msg)


def window(**kw):
    a = dict(q=P, out=P, kc=P, vc=P, seq=P, n=P, tab=P, cu=None, seqs=2, tokens=4, qh=8, kvh=4, hd=128, bs=64, mb=4,
             blocks=9, scale=0.1, window=10, sinks=2, stride=1024, mql=0, ws=None, wb=0, dt=1)
    a.update(kw)
    return ops.lib().nvf_window_attention_ws(*a.values(), None)


def test_window_attention_refusals():
    for kw, text in ((dict(dt=3), "dtype"), (dict(tokens=-1), "shape"), (dict(kvh=3), "multiple"), (dict(hd=257), "256"),
                     (dict(bs=0), "shape"), (dict(stride=1023), "q_stride"), (dict(out=None), "NULL"),
                     (dict(tab=None), "NULL"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
                     (dict(ws=P + 4, wb=99), "workspace"), (dict(seqs=-1), "shape"), (dict(blocks=-1), "shape"),
                     (dict(blocks=0), "shape"), (dict(bs=1 << 20, mb=1 << 12), "2^31"),
                     (dict(tokens=1 << 40), "many")):
        refused(window(**kw), text)
    for cu in ([1, 2, 4], [0, 2, 3], [0, 5, 4]):
        a = np.array(cu, np.int32)
        refused(window(cu=a.ctypes.data), "cu_seqlens")
    assert window(tokens=0, q=None) == 0
    size = ops.lib().nvf_window_attention_workspace_size
    assert size(0, 8, 4, 128, 64, 4, 10, 2, 1) == 0 and size(4, 8, 3, 128, 64, 4, 10, 2, 1) == 0


def prefix(start=(0, 4), lens=(10,), **kw):
    s, n = np.array(start, np.int32), np.array(lens, np.int32)
    a = dict(q=P, out=P, kc=P, vc=P, seq=P, n=P, tab=P, start=s.ctypes.data, lens=n.ctypes.data, groups=len(n), seqs=2,
             tokens=4, qh=8, kvh=4, hd=128, bs=64, mb=4, blocks=9, scale=0.1, stride=1024, ws=None, wb=0, dt=1)
    a.update(kw)
    return ops.lib().nvf_prefix_attention_ws(*a.values(), None)


def test_prefix_attention_refusals():
    for kw, text in ((dict(dt=3), "dtype"), (dict(kvh=3), "multiple"), (dict(q=None), "NULL"), (dict(groups=0), "groups"),
                     (dict(start=(0, 3)), "group_start"), (dict(start=(1, 4)), "group_start"),
                     (dict(start=(0, 5, 4), lens=(1, 1)), "decrease"), (dict(lens=(-1,)), "prefix_len"),
                     (dict(lens=(257,)), "prefix_len"), (dict(ws=P + 8, wb=9), "workspace")):
        refused(prefix(**kw), text)
    assert prefix(start=(0, 0), tokens=0) == 0


def test_page_refusals():
    lib = ops.lib()
    caches = (C.c_void_p * 2)(1 << 20, 2 << 20)
    ints = lambda *v: np.array(v, np.int32)  # noqa: E731

    def copy(src, dst, n_caches=2, n=None, pages=10, page_bytes=64, c=caches):
        s, d = ints(*src), ints(*dst)
        return lib.nvf_copy_pages(c, n_caches, s.ctypes.data, d.ctypes.data, len(s) if n is None else n, pages, page_bytes,
                                  None)

    refused(copy([0], [10]), "outside")
    refused(copy([-1], [1]), "outside")
    refused(copy([10], [1]), "outside")
    refused(copy([0, 1], [2, 2]), "twice")
    refused(copy([0, 1], [1, 2]), "source")
    refused(copy([3], [3]), "source")
    refused(copy([0], [1], n=-1), "number")
    refused(copy([0], [1], page_bytes=0), "shape")
    refused(copy([0], [1], page_bytes=1 << 50), "shape")
    refused(copy([0], [1], pages=-1), "shape")
    refused(copy([0], [1], c=(C.c_void_p * 2)(1 << 20, None)), "NULL")
    refused(copy([0], [1], c=(C.c_void_p * 2)(1 << 20, (1 << 20) + 64)), "overlap")
    assert copy([], []) == 0 and copy([0], [1], n_caches=0) == 0

    def fork(parent, child, rows=8, cols=4, pages=10, bs=16, row_bytes=4, tab=P, n_caches=2):
        p, c = ints(*parent), ints(*child)
        return lib.nvf_fork_pages(caches, n_caches, tab, P, P, p.ctypes.data, c.ctypes.data, len(p), P, rows, cols, pages,
                                  bs, row_bytes, None)

    refused(fork([0], [0]), "parent and a child")
    refused(fork([0, 1], [2, 2]), "twice")
    refused(fork([0, 2], [2, 3]), "parent and a child")
    refused(fork([8], [1]), "outside")
    refused(fork([1], [-1]), "outside")
    refused(fork([1], [2], bs=0), "shape")
    refused(fork([1], [2], cols=0), "shape")
    refused(fork([1], [2], tab=None), "NULL")
    assert fork([], []) == 0

    def free(seqs, window=-1, sinks=0, rows=8, bs=16):
        s = ints(*seqs)
        return lib.nvf_free_pages(P, P, P, s.ctypes.data, len(s), rows, 4, 10, bs, window, sinks, None)

    refused(free([8]), "outside")
    refused(free([1, 1]), "twice")
    refused(free([1], sinks=-1), "shape")
    refused(free([1], bs=0), "shape")
    assert free([]) == 0

    def compact(wb=1 << 20, ws=P, ref=P, entries_ptr=P, page_bytes=64):
        return lib.nvf_compact_pages(caches, 2, entries_ptr, ref, P, P, None, 8, 4, 10, page_bytes, ws, wb, None)

    refused(compact(wb=100), "workspace")
    refused(compact(ws=None), "NULL")
    refused(compact(ref=None), "NULL")
    refused(compact(entries_ptr=None), "NULL")
    refused(compact(page_bytes=-1), "shape")
    assert lib.nvf_compact_pages_workspace_size(10) == 124 and lib.nvf_compact_pages_workspace_size(-1) == 0


def rotary(**kw):
    a = dict(q=1 << 20, q_out=1 << 20, k=2 << 20, k_out=2 << 20, v=None, pos=P, freq=P, inter=0, rot=64, scale=1.0,
             qw=None, kw=None, eps=1e-6, tokens=4, qh=8, kvh=4, hd=128, qs=1024, qos=1024, ks=512, kos=512, vs=0, kc=None,
             vc=None, slots=None, rows=0, dt=1)
    a.update(kw)
    return ops.lib().nvf_rotary(*a.values(), None)


def test_rotary_refusals():
    q = 1 << 20
    for kw, text in ((dict(dt=-1), "dtype"), (dict(hd=258), "shape"), (dict(rot=63), "even part"), (dict(rot=130), "even part"),
                     (dict(qs=1000), "stride"), (dict(kos=100), "stride"), (dict(qw=P), "together"),
                     (dict(kc=P), "store"), (dict(kc=P, vc=P, v=P, vs=512), "store"), (dict(k_out=None), "NULL"),
                     (dict(pos=None), "NULL"), (dict(freq=None), "NULL"), (dict(q_out=q + 2), "overlaps q"),
                     (dict(q_out=q + 2048, qos=2048), "overlaps q"), (dict(q_out=2 << 20), "overlaps k"),
                     (dict(k_out=q + 1024, kos=512), "overlaps q"), (dict(q_out=3 << 20, k_out=3 << 20), "q_out overlaps k_out"),
                     # columns of one packed row that cross
                     (dict(qs=4096, q_out=q + 1024, qos=4096), "overlaps q"), (dict(tokens=1 << 31), "many")):
        refused(rotary(**kw), text)
    assert rotary(tokens=0) == 0


def test_python_refusals():
    """Shapes, types and places are checked before any call."""
    t = torch.zeros
    q, kc = t(3, 8, 64), t(32, 2, 64)
    meta = t(3, dtype=torch.int32), t(3, dtype=torch.int32), t(2, 2, dtype=torch.int32)
    for call in (lambda **k: ops.window_attention(**{**base, **k}, window=4),
                 lambda **k: ops.prefix_attention(**{**base, **k}, prefix_len=4)):
        base = dict(q=q, k_cache=kc, v_cache=kc, query_seq=meta[0], query_key_len=meta[1], block_tables=meta[2],
                    block_size=16, scale=0.1)
        with pytest.raises(ValueError, match="GPU tensor"):
            call()
        for kw in (dict(q=q[0]), dict(k_cache=t(32, 2, 32)), dict(v_cache=t(16, 2, 64)), dict(v_cache=kc.half()),
                   dict(query_seq=meta[0][:2]), dict(query_key_len=meta[1].long()), dict(block_tables=meta[0]),
                   dict(block_size=0), dict(block_size=15), dict(out=t(3, 8, 32)), dict(out=q.half()),
                   dict(block_tables=meta[2][:, :0])):
            with pytest.raises(ValueError):
                call(**kw)
    with pytest.raises(ValueError, match="whole numbers"):
        ops.copy_pages([], [0.5], [1], 16)
    with pytest.raises(ValueError, match="32 bits"):
        ops.copy_pages([], [2 ** 40], [1], 16)
    with pytest.raises(ValueError, match="one length"):
        ops.copy_pages([], [0], [1, 2], 16)
    with pytest.raises(ValueError, match="one shape"):
        ops.copy_pages([kc, kc.half()], [0], [1], 16)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.copy_pages([kc], [0], [1], 16)
    with pytest.raises(ValueError, match="ref_count"):
        ops.free_pages(meta[2], meta[0][:2], meta[0].long(), [0], 16)
    with pytest.raises(ValueError, match="key_len"):
        ops.free_pages(meta[2], meta[0], meta[0], [0], 16)
    x, pos, f = t(3, 512), t(3, dtype=torch.int64), t(32, dtype=torch.float64)
    for kw in (dict(positions=pos.int()), dict(inv_freq=f.float()), dict(inv_freq=t(33, dtype=torch.float64)),
               dict(k=t(3, 64)), dict(q_out=t(3, 500)), dict(q_w=t(32)), dict(k=x[:, :128].half())):
        with pytest.raises(ValueError):
            ops.rotary(**{**dict(q=x, k=x[:, :128], positions=pos, inv_freq=f, q_heads=8, kv_heads=2, head_dim=64), **kw})
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.rotary(x, x[:, :128], pos, f, 8, 2, 64)


def test_rotary_inv_freq():
    """The tables by their definitions (double: equal to a few units)."""
    d, theta, L = 128, 1e6, 8192.0
    i = np.arange(d // 2)
    f = theta ** (-2.0 * i / d)
    plain, s = ops.rotary_inv_freq(theta, d)
    assert np.allclose(plain.numpy(), f, rtol=1e-14) and s == 1.0
    assert np.allclose(plain.numpy().astype(np.float32), ops.rope_inv_freq(theta, d).numpy(), rtol=1e-7)
    linear, s = ops.rotary_inv_freq(theta, d, ops.ROPE_LINEAR, 4.0)
    assert np.allclose(linear.numpy(), f / 4, rtol=1e-14) and s == 1.0
    turns = L * f / (2 * math.pi)
    ramp, s = ops.rotary_inv_freq(theta, d, ops.ROPE_RAMP, 4.0, 1.0, 32.0, L)
    at = [d * math.log(L / (n * 2 * math.pi)) / (2 * math.log(theta)) for n in (32.0, 1.0)]
    lo, hi = math.floor(at[0]), math.ceil(at[1])
    keep = 1 - np.clip((i - lo) / (hi - lo), 0, 1)
    assert np.allclose(ramp.numpy(), f * keep + f / 4 * (1 - keep), rtol=1e-13)
    assert abs(s - (0.1 * math.log(4.0) + 1)) < 1e-7
    assert np.allclose(ramp.numpy()[turns > 40], f[turns > 40]) and np.allclose(ramp.numpy()[turns < 0.8], f[turns < 0.8] / 4)
    bands, s = ops.rotary_inv_freq(theta, d, ops.ROPE_BANDS, 8.0, 1.0, 4.0, L)
    keep = np.clip((turns - 1) / 3, 0, 1)
    assert np.allclose(bands.numpy(), f * keep + f / 8 * (1 - keep), rtol=1e-13) and s == 1.0
    for bad in ((0.0, 64), (1e4, 63), (1e4, 0), (1e4, 64, 9), (1e4, 64, 1, 0.5), (1e4, 64, 2, 2.0, 2.0, 1.0, 100.0),
                (1e4, 64, 2, 2.0, 1.0, 32.0, 0.0), (1.0, 64, 2, 2.0, 1.0, 32.0, 100.0), (float("nan"), 64)):
        with pytest.raises(ops.NvfError):
            ops.rotary_inv_freq(*bad)
