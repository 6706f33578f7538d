"""Refusals of the 4-bit cache's operators and of prompt attention (host only: no call here reaches a launch), and the
cache's rows against hand-worked ones."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from nano_vllm_cpp_amd import ops
from tests import kv4

P = 0x1000  # never dereferenced


def refused(rc, text):
    msg = ops.lib().nvf_last_error().decode()
    assert rc == -1 and text in msg, (rc, msg)


def test_row_bytes():
    assert ops.kv4_row_bytes(4, 128) == 288 and ops.kv4_row_bytes(2, 64) == 80 and ops.kv4_row_bytes(1, 32) == 32
    for kvh, hd in ((0, 64), (4, 48), (4, 288), (4, 0), (-1, 64)):
        assert ops.lib().nvf_kv4_row_bytes(kvh, hd) == 0
        with pytest.raises(ValueError):
            ops.kv4_row_bytes(kvh, hd)
    for kvh in range(1, 9):
        for hd in range(32, 257, 32):
            assert ops.kv4_row_bytes(kvh, hd) == kv4.row_bytes(kvh, hd)


def test_definition():
    """A group by hand: -3 .. 4.5 takes d = 0.5 and z = 6."""
    x = np.zeros((1, 1, 32))
    x[0, 0, :6] = [-3.0, 4.5, 0.25, 0.75, -0.25, 4.0]
    codes, words = kv4.quantize(x)
    assert codes[0, 0, :6].tolist() == [0, 15, 6, 8, 6, 14] and (codes[0, 0, 6:] == 6).all()  # (ties to even)
    assert words[0, 0].tolist() == [0x3800 | 6]
    back = kv4.values(kv4.pack(codes, words), 1, 32)
    assert back[0, 0, :6].tolist() == [-3.0, 4.5, 0.0, 1.0, 0.0, 4.0]
    zero = kv4.quantize(np.zeros((1, 1, 32)))
    assert (zero[0] == 0).all() and (zero[1] == 0).all()
    x[0, 0, 9] = np.inf
    assert (kv4.quantize(x)[1] == 0x7E00).all() and np.isnan(kv4.values(kv4.pack(*kv4.quantize(x)), 1, 32)).all()


def store(**kw):
    a = dict(q=P, qo=P, k=P << 20, ko=None, v=P << 22, pos=P, f=P, il=0, rot=64, s=1.0, qw=None, kw=None, eps=1e-6,
             tokens=4, qh=8, kvh=4, hd=128, qs=1024, qos=1024, ks=512, kos=512, vs=512, kc=P << 24, vc=P << 26, slots=P,
             rows=100, dt=1)
    a.update(kw)
    return ops.lib().nvf_rotary_store_kv4(*a.values(), None)


def test_store_refusals():
    for kw, text in ((dict(dt=3), "dtype"), (dict(tokens=-1), "shape"), (dict(hd=80), "multiple of 32"), (dict(hd=288), "256"),
                     (dict(rot=63), "even part"), (dict(rot=130), "even part"), (dict(qs=1023), "stride"),
                     (dict(vs=511), "stride"), (dict(ko=P << 21, kos=511), "stride"), (dict(qw=P), "together"),
                     (dict(kc=None), "NULL"), (dict(vc=None), "store needs"), (dict(slots=None), "store needs"),
                     (dict(v=None), "store needs"), (dict(q=None), "NULL"), (dict(pos=None), "NULL"),
                     (dict(kc=(P << 24) + 8), "aligned"), (dict(vc=(P << 24) + 16), "overlaps"), (dict(rows=-1), "shape"),
                     (dict(qo=P << 20), "overlaps"), (dict(ko=P << 22), "overlaps"), (dict(tokens=1 << 40), "many"),
                     (dict(kvh=0, ks=0), "store needs")):
        refused(store(**kw), text)
    assert store(tokens=0) == 0 and store(tokens=0, q=None, kc=None) == 0


def unpack(**kw):
    a = dict(cache=P, out=P << 20, rows=10, kvh=4, hd=128, dt=1)
    a.update(kw)
    return ops.lib().nvf_kv4_unpack(*a.values(), None)


def test_unpack_refusals():
    for kw, text in ((dict(dt=7), "dtype"), (dict(rows=-1), "shape"), (dict(hd=48), "shape"), (dict(kvh=0), "shape"),
                     (dict(cache=None), "NULL"), (dict(out=None), "NULL"), (dict(cache=P + 8), "aligned"),
                     (dict(out=P + 4), "aligned"), (dict(out=P + 1024), "overlaps"), (dict(rows=1 << 50), "many")):
        refused(unpack(**kw), text)
    assert unpack(rows=0, cache=None) == 0


def paged(**kw):
    a = dict(q=P, out=P, kc=P, vc=P, seq=P, n=P, tab=P, cu=None, seqs=2, tokens=4, qh=8, kvh=4, hd=128, bs=64, mb=4,
             blocks=9, scale=0.1, stride=1024, mql=0, ws=None, wb=0, dt=1)
    a.update(kw)
    return ops.lib().nvf_paged_attention_kv4_ws(*a.values(), None)


def test_paged_refusals():
    for kw, text in ((dict(dt=3), "dtype"), (dict(tokens=-1), "shape"), (dict(kvh=3), "multiple"), (dict(hd=288), "256"),
                     (dict(hd=80), "multiple of 32"), (dict(bs=0), "shape"), (dict(stride=1023), "q_stride"),
                     (dict(out=None), "NULL"), (dict(tab=None), "NULL"), (dict(ws=P + 4, wb=99), "workspace"),
                     (dict(seqs=-1), "shape"), (dict(blocks=0), "shape"), (dict(bs=1 << 20, mb=1 << 12), "2^31"),
                     (dict(tokens=1 << 40), "many"), (dict(kc=P + 8), "aligned"), (dict(vc=P + 4), "aligned")):
        refused(paged(**kw), text)
    for cu in ([1, 2, 4], [0, 2, 3], [0, 5, 4]):
        a = np.array(cu, np.int32)
        refused(paged(cu=a.ctypes.data), "cu_seqlens")
    assert paged(tokens=0, q=None) == 0
    size = ops.lib().nvf_paged_attention_kv4_workspace_size
    assert size(0, 8, 4, 128, 64, 4, 1) == 0 and size(4, 8, 3, 128, 64, 4, 1) == 0 and size(4, 8, 4, 80, 64, 4, 1) == 0


def prompt(**kw):
    a = dict(q=P, k=P << 12, v=P << 16, out=P << 20, cu=P, seqs=2, tokens=4, qh=8, kvh=4, hd=128, scale=0.1, qs=1024,
             ks=512, vs=512, ws=None, wb=0, dt=1)
    a.update(kw)
    return ops.lib().nvf_prompt_attention_ws(*a.values(), None)


def test_prompt_refusals():
    for kw, text in ((dict(dt=-1), "dtype"), (dict(tokens=-1), "shape"), (dict(seqs=-1), "shape"), (dict(kvh=3), "multiple"),
                     (dict(hd=257, qs=9999, ks=9999, vs=9999), "256"), (dict(qs=1023), "stride"), (dict(ks=511), "stride"),
                     (dict(vs=511), "stride"), (dict(ws=P + 8, wb=9), "workspace"), (dict(q=None), "NULL"),
                     (dict(cu=None), "NULL"), (dict(out=P + 1024), "overlaps"), (dict(out=(P << 12) + 64), "overlaps"),
                     (dict(out=(P << 16) + 64), "overlaps"), (dict(tokens=1 << 40), "many")):
        refused(prompt(**kw), text)
    assert prompt(tokens=0, q=None) == 0 and prompt(seqs=0, cu=None) == 0
    size = ops.lib().nvf_prompt_attention_workspace_size
    assert size(1, 0, 8, 4, 128) == 0 and size(0, 9, 8, 4, 128) == 0 and size(1, 9, 8, 3, 128) == 0


def test_front_end_refusals():
    """Shapes, types and devices that the front end refuses before the library sees them."""
    t, qh, kvh, hd, bs = 4, 8, 4, 64, 16
    q = torch.zeros((t, qh, hd), dtype=torch.float16)
    row = ops.kv4_row_bytes(kvh, hd)
    kc = torch.zeros((2 * bs, row), dtype=torch.uint8)
    ints = torch.zeros(t, dtype=torch.int32)
    table = torch.zeros((t, 2), dtype=torch.int32)

    def attend(q=q, kc=kc, vc=None, kvh=kvh, seq=ints, n=ints, table=table, bs=bs, **kw):
        return ops.paged_attention_kv4(q, kc, kc if vc is None else vc, kvh, seq, n, table, bs, 0.1, **kw)

    for kw, text in ((dict(), "GPU tensor"), (dict(q=q[0]), "q must be"), (dict(kvh=3), "k_cache and v_cache"),
                     (dict(kc=kc[:, :-1]), "k_cache and v_cache"), (dict(vc=kc[:bs]), "k_cache and v_cache"),
                     (dict(kc=kc.to(torch.int8)), "k_cache and v_cache"), (dict(seq=ints.long()), "query_seq"),
                     (dict(n=ints[:2]), "query_key_len"), (dict(table=table[0]), "block_tables"), (dict(bs=24), "whole blocks"),
                     (dict(out=q.float()), "out must"), (dict(q=torch.zeros((t, qh, 48))), "multiple of 32")):
        with pytest.raises(ValueError, match=text):
            attend(**kw)
    k = torch.zeros((t, kvh, hd), dtype=torch.float16)
    cu = torch.tensor([0, t], dtype=torch.int32)
    for args, kw, text in (((q, k, k, cu), {}, "GPU tensor"), ((q, k[:2], k[:2], cu), {}, "q must be"),
                           ((q, k, k.float(), cu), {}, "dtype"), ((q, k, k, cu.long()), {}, "cu_seqlens"),
                           ((q, k, k, cu[:0]), {}, "cu_seqlens"), ((q, k, k, cu), dict(out=q.float()), "out must")):
        with pytest.raises(ValueError, match=text):
            ops.prompt_attention(*args, 0.1, **kw)
    with pytest.raises(ValueError, match="uint8"):
        ops.kv4_unpack(kc[:, :-1], kvh, hd)
    with pytest.raises(ValueError, match="out must"):
        ops.kv4_unpack(kc, kvh, hd, out=torch.zeros((2 * bs, kvh, hd)))
    pos, f = torch.zeros(t, dtype=torch.int64), torch.zeros(hd // 2, dtype=torch.float64)
    rows = [torch.zeros((t, n * hd), dtype=torch.float16) for n in (qh, kvh, kvh)]
    for kw, text in ((dict(), "GPU tensor"), (dict(slots=ints.long()), "slot_mapping"), (dict(kc=kc[:, 1:]), "k_cache and"),
                     (dict(pos=pos.int()), "positions"), (dict(q_w=torch.ones(hd)), "q_w")):
        a = dict(pos=pos, kc=kc, slots=ints)
        a.update({n: kw.pop(n) for n in list(kw) if n in a})
        with pytest.raises(ValueError, match=text):
            ops.rotary_store_kv4(*rows, a["pos"], f, qh, kvh, hd, a["kc"], a["kc"], a["slots"], **kw)
