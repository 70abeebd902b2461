"""The tree operators' C entry points refuse bad arguments with a status before they touch the device, and the
64-bit restatement of the operators agrees with small cases worked by hand."""

import ctypes

import numpy as np
import pytest

from myinfer_b200 import _lib
from oracle import tree as ref

P = ctypes.c_void_p(16)
I3 = (ctypes.c_int64 * 3)(1024, 128, 128)


def _attention(**kw):
    v = _lib.M5KvView(16, 16, 16, 0, 100)
    a = dict(q=P, qs=I3, B=1, Hq=8, L=4, D=128, k=v, v=v, Hkv=2, cap=100, lengths=P, T=4, anc=P, anc_s=4, scale=1.0,
             group=64, bits=8, out=P, os=I3, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    rc = _lib.lib().m5_tree_attention(*a.values())
    return rc, _lib.last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(q=None), "null"), (dict(qs=None), "null"), (dict(lengths=None), "null"), (dict(anc=None), "null"),
    (dict(L=0), "empty"), (dict(cap=0), "empty"), (dict(Hkv=3), "multiple"), (dict(D=96), "head_dim"),
    (dict(L=65), "64 nodes"), (dict(T=65), "64 nodes"), (dict(bits=3), "bits"), (dict(group=32), "group_size"),
    (dict(cap=2 ** 31), "capacity"), (dict(k=_lib.M5KvView(24, 16, 16, 0, 100)), "aligned"),
    (dict(k=_lib.M5KvView(16, None, 16, 0, 100)), "scales"), (dict(qs=(ctypes.c_int64 * 3)(1024, 128, 4)), "aligned"),
    (dict(out=ctypes.c_void_p(24)), "aligned")])
def test_attention_refusals(kw, text):
    rc, msg = _attention(**kw)
    assert rc == _lib.M5_ERR_INVALID and text in msg, msg


def test_other_refusals():
    L = _lib.lib()
    bad = _lib.M5_ERR_INVALID
    assert L.m5_tree_plan(None, 1, 4, P, None, None) == bad
    assert L.m5_tree_plan(P, 1, 65, P, None, None) == bad and "64" in _lib.last_error()
    assert L.m5_tree_accept(P, P, P, 0, 4, P, P, P, None, 0, 0, None) == bad
    assert L.m5_tree_accept(P, P, P, 1, 4, P, P, P, P, 5, 9, None) == bad and "counts" in _lib.last_error()
    ly = (_lib.M5LayerKv * 1)(_lib.M5LayerKv(16, 16, 16, 16, 16, 16, 64, 3, 64))
    assert L.m5_tree_commit(ly, 1, 1, 1, 128, P, P, 4, P, None) == bad and "bits" in _lib.last_error()
    ly[0].bits, ly[0].v_scales = 8, None
    assert L.m5_tree_commit(ly, 1, 1, 1, 128, P, P, 4, P, None) == bad and "scales" in _lib.last_error()
    assert L.m5_tree_commit(ly, 1, 1, 1, 96, P, P, 4, P, None) == bad
    n = ctypes.c_size_t(0)
    assert L.m5_tree_attention_workspace(1, 7, 2, 4, 128, ctypes.byref(n)) == bad

    def logits(**kw):
        a = dict(x=P, ld=100, out=P, old=100, dt=0, B=2, T=3, V=100, counts=None, cld=0, pen=None, tok=None, anc=None,
                 ids=None, val=None, nb=0, mask=None, mld=0, ch=None, st=None)
        a.update(kw)
        return L.m5_process_logits(*a.values())
    for kw, text in ((dict(x=None), "null"), (dict(dt=7), "dtype"), (dict(V=0), "empty"), (dict(T=65), "64"),
                     (dict(V=600000, ld=600000, old=600000), "vocabulary"), (dict(ld=99), "stride"),
                     (dict(counts=P, cld=100), "penalties"), (dict(tok=P, pen=P), "ancestors"),
                     (dict(nb=1025, ids=P, val=P), "bias"), (dict(nb=3), "bias"), (dict(mask=P, mld=3), "mask"),
                     (dict(B=2000, T=64), "rows")):
        assert logits(**kw) == bad and text in _lib.last_error(), kw


def test_restatement():
    p = np.array([[-1, 0, 0, 1, 3, 5, -1]], np.int32)  # node 5 is no earlier node of itself: no node
    bits, depth = ref.ancestors(p)
    assert bits[0].tolist() == [1, 3, 5, 11, 27, 0, 64] and depth[0].tolist() == [0, 1, 1, 2, 3, 0, 0]
    assert ref.accept([-1, 0, 0, 2], [9, 4, 5, 6], [5, 1, 6, 2]) == ([0, 2, 3], 2)
    assert ref.accept([-1, 0, 0], [9, 4, 4], [4, 8, 7]) == ([0, 1], 8)
    y = ref.process_row(np.array([2.0, -2.0, 1.0, 0.5]), np.array([1, 0, 0, 0]), (2.0, 0.25, 0.5), [1, 1], [(2, 1), (2, 3)],
                        [0b0111])
    assert y.tolist() == [2 / 2 - 0.25 - 0.5, -4 - 0.25 - 1.0, 4.0, -np.inf] and ref.choice(y) == 2
    q = np.ones((1, 1, 2))
    k = np.zeros((1, 3, 2))
    v = np.array([[[1.0, 2.0], [3.0, 4.0], [9.0, 9.0]]])
    out, _ = ref.attention(q, k, v, 1, [1], 1, 1.0)
    assert out[0, 0].tolist() == [2.0, 3.0]
    assert (ref.attention(q, k, v, 0, [0], 1, 1.0)[0] == 0).all()
