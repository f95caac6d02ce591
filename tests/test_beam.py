"""What the operators of decoding with beams refuse, on the host (no GPU needed)."""
import ctypes

import pytest
import torch

import asrq_b200
from asrq_b200 import _lib

I3 = ctypes.c_int64 * 3


def _ptr(n=64):
    buf = ctypes.create_string_buffer(n + 16)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def _select(**kw):
    keep, p = _ptr()
    a = dict(logits=p, sb=10, sk=10, scores=p, finished=None, eos=0, out=p, parents=p, tokens=p, out_finished=None, B=1, K=2, V=10, n=2, dtype=0)
    a.update(kw)
    return _lib.load().asrq_beam_select(a["logits"], a["sb"], a["sk"], a["scores"], a["finished"], a["eos"], a["out"], a["parents"], a["tokens"], a["out_finished"],
                                        a["B"], a["K"], a["V"], a["n"], a["dtype"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(logits=None), -1), (dict(scores=None), -1), (dict(out=None), -1), (dict(parents=None), -1), (dict(tokens=None), -1), (dict(finished=1), -1),
    (dict(dtype=2), -5), (dict(B=-1), -2), (dict(K=0), -2), (dict(V=0), -2), (dict(n=0), -2), (dict(n=21), -2), (dict(sk=-1), -2),
    (dict(finished=1, out_finished=1, eos=10), -2), (dict(finished=1, out_finished=1, eos=-1), -2), (dict(K=33), -8), (dict(K=4, V=100, n=33), -8),
    (dict(K=32, V=65536 * 4 + 1), -8), (dict(K=1, V=65536 * 128 + 1, n=1), -8), (dict(logits=17), -3),
])
def test_select_refusals(kw, code):
    assert _select(**kw) == code
    assert "asrq_beam_select" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(cache=None), -1), (dict(parents=None), -1), (dict(K=0), -2), (dict(bytes=24), -2), (dict(bytes=0), -2), (dict(L=-1), -2), (dict(heads=0), -2),
    (dict(max_len=0), -2), (dict(K=33), -8), (dict(odd=2), -3), (dict(ws=None), -4), (dict(ws_bytes=255), -4),
])
def test_reorder_refusals(kw, code):
    keep, p = _ptr()
    a = dict(cache=p, parents=p, L=1, B=1, K=2, heads=1, max_len=4, bytes=16, odd=0, ws=p, ws_bytes=256)
    a.update(kw)
    rc = _lib.load().asrq_beam_reorder(a["cache"] and a["cache"] + a["odd"], a["parents"], None, 2, a["L"], a["B"], a["K"], a["heads"], a["max_len"], a["bytes"], a["ws"], a["ws_bytes"], None)
    assert rc == code and "asrq_beam_reorder" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(out=None), -1), (dict(dtype=2), -5), (dict(hd=96), -2), (dict(nq=3), -2), (dict(nkv=0), -2), (dict(keys=-1), -2),
    (dict(B=-1), -2), (dict(R=-1), -2), (dict(qs=I3(8, 8, 4)), -3), (dict(ks=I3(8, -8, 8)), -3), (dict(odd=2), -3), (dict(scratch=24), -3),
])
def test_cross_refusals(kw, code):
    keep, p = _ptr()
    s = I3(64, 64, 64)
    a = dict(q=p, k=p, v=p, out=p, qs=s, ks=s, B=1, R=1, nq=2, nkv=2, hd=64, keys=4, dtype=0, odd=0, scratch=None)
    a.update(kw)
    rc = _lib.load().asrq_cross_attention(a["q"] and a["q"] + a["odd"], a["qs"], a["k"], a["ks"], a["v"], s, None, a["out"], a["B"], a["R"], a["nq"], a["nkv"], a["hd"],
                                          a["keys"], 1.0, a["dtype"], None, 0, a["scratch"], 0, None)
    assert rc == code and "asrq_cross_attention" in _lib.last_error()


@pytest.mark.parametrize("kw,code", [(dict(lengths=None), -1), (dict(n=3), -2), (dict(n=0), -2), (dict(ks=None), -1), (dict(hd=32), -2), (dict(suffix=-1), -2)])
def test_prefix_refusals(kw, code):
    keep, p = _ptr()
    s = I3(64, 64, 64)
    a = dict(lengths=p, n=1, ks=p, hd=64, suffix=4)
    a.update(kw)
    rc = _lib.load().asrq_prefix_attention(p, s, p, s, p, s, None, a["ks"], s, p, s, a["lengths"], a["n"], p, 1, 2, 2, 2, a["hd"], 4, a["suffix"], 1.0, 0, None, 0, None, 0, None)
    assert rc == code and "asrq_prefix_attention" in _lib.last_error()


def test_no_cpu_path():
    x = torch.zeros(1, 2, 10, dtype=torch.float16)
    q = torch.zeros(1, 2, 2, 64, dtype=torch.float16)
    n = torch.zeros(1, dtype=torch.int64)
    for call in (lambda: asrq_b200.beam_select(x, torch.zeros(1, 2)), lambda: asrq_b200.cross_attention(q, q, q),
                 lambda: asrq_b200.prefix_attention(q, q, q, q, q, n), lambda: asrq_b200.beam_reorder(torch.zeros(1, 2, 1, 4, 8), torch.zeros(1, 2, dtype=torch.int64), 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
