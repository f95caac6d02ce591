"""The ways to call the operators of decoding with beams: both host paths, other streams, threads, no scratch, unusual strides."""
import threading

import pytest
import torch

import asrq_b200
from asrq_b200 import _lib, linear
from tests.beam_util import check_rows, check_select

DEV = "cuda"
pytestmark = pytest.mark.gpu


def _rnd(seed, *shape, dtype=torch.float16, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


def _calls():
    logits, scores, over = _rnd(1, 2, 3, 999, std=3), _rnd(2, 2, 3, dtype=torch.float32), torch.tensor([[False, True, False], [True, False, False]], device=DEV)
    parents, cache = torch.tensor([[1, 1, 0], [2, 0, 1]], device=DEV), _rnd(3, 4, 6, 2, 9, 64)
    q, kv, lengths = _rnd(4, 2, 40, 4, 64), _rnd(5, 2, 300, 2, 2, 64), torch.tensor([300, 7], device=DEV)
    own, n_own = _rnd(6, 80, 2, 12, 64), torch.arange(80, device=DEV) % 13
    return {
        "select": lambda: asrq_b200.beam_select(logits, scores, 5),
        "select, ended": lambda: asrq_b200.beam_select(logits, scores, 5, finished=over, eos=7),
        "reorder": lambda: (asrq_b200.beam_reorder(cache.clone(), parents, 7),),
        "reorder, on the device": lambda: (asrq_b200.beam_reorder(cache.clone(), parents, torch.tensor([8], device=DEV)),),
        "cross": lambda: (asrq_b200.cross_attention(q, kv[:, :, 0], kv[:, :, 1], lengths),),
        "prefix": lambda: (asrq_b200.prefix_attention(q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), own, own, n_own, lengths),),
    }


@pytest.mark.parametrize("name", sorted(["select", "select, ended", "reorder", "reorder, on the device", "cross", "prefix"]))
def test_both_host_paths_and_another_stream(name, monkeypatch):
    call = _calls()[name]
    first = call()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        second = call()
        torch.cuda.current_stream().synchronize()
    monkeypatch.setattr(linear, "_native", None)
    third = call()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(first, second, third))
    asrq_b200.check_status()


def test_two_threads_on_streams_of_their_own():
    calls = _calls()
    want = {k: f() for k, f in calls.items()}
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                for k, f in calls.items():
                    got = f()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[k])):
                        wrong.append(k)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    asrq_b200.check_status()


@pytest.mark.parametrize("offset", range(8))
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 15, 16, 23, 1023, 1025, 4097])
def test_select_reads_its_rows_and_nothing_else(V, offset):
    """Rows at every alignment, what lies around them infinite."""
    B, K, n = 2, 3, min(3 * V, 6)
    flat = torch.full((offset + B * K * (V + 3) + 16,), float("inf"), dtype=torch.float16, device=DEV)
    logits = flat[offset:offset + B * K * (V + 3)].view(B, K, V + 3)[:, :, :V]
    logits.copy_(_rnd(V + offset, B, K, V, std=3))
    scores = _rnd(offset, B, K, dtype=torch.float32)
    check_select(asrq_b200.beam_select(logits, scores, n), logits, scores, n)


def _strides(x, *dims):
    return asrq_b200.beam._strides(x, *dims)


@pytest.mark.parametrize("R", [5, 150])
@pytest.mark.parametrize("memory", ["none", "workspace", "too little"])
def test_without_scratch(R, memory):
    """The C entry points without the memory that dividing the keys takes, or with too little of it: the kernels that need none."""
    B, S, M, H, hd = 1, 700, 20, 2, 64
    q, k, v = _rnd(1, B, R, H, hd), _rnd(2, B, H, S, hd), _rnd(3, B, H, S, hd)
    k2, v2, n2 = _rnd(4, B * R, H, M, hd), _rnd(5, B * R, H, M, hd), torch.arange(B * R, device=DEV) % (M + 1)
    ws = torch.zeros(_lib.STATUS_BYTES, dtype=torch.uint8, device=DEV)
    scratch = torch.zeros(64, dtype=torch.uint8, device=DEV)
    memory = {"none": (None, 0, None, 0), "workspace": (ws.data_ptr(), ws.numel(), None, 0), "too little": (ws.data_ptr(), ws.numel(), scratch.data_ptr(), 64)}[memory]
    stream = torch.cuda.current_stream().cuda_stream
    out = torch.empty_like(q)
    _lib.call("asrq_cross_attention", q.data_ptr(), _strides(q, 0, 1, 2), k.data_ptr(), _strides(k, 0, 1, 2), v.data_ptr(), _strides(v, 0, 1, 2), None, out.data_ptr(),
              B, R, H, H, hd, S, hd ** -0.5, _lib.F16, *memory, stream)
    check_rows(out, q, lambda b, r: (k[b].transpose(0, 1), v[b].transpose(0, 1)))
    _lib.call("asrq_prefix_attention", q.data_ptr(), _strides(q, 0, 1, 2), k.data_ptr(), _strides(k, 0, 1, 2), v.data_ptr(), _strides(v, 0, 1, 2), None,
              k2.data_ptr(), _strides(k2, 0, 1, 2), v2.data_ptr(), _strides(v2, 0, 1, 2), n2.data_ptr(), B * R, out.data_ptr(), B, R, H, H, hd, S, M, hd ** -0.5,
              _lib.F16, *memory, stream)
    n = n2.tolist()
    check_rows(out, q, lambda b, r: (torch.cat((k[b].transpose(0, 1), k2[r, :, :n[r]].transpose(0, 1))), torch.cat((v[b].transpose(0, 1), v2[r, :, :n[r]].transpose(0, 1)))))
    assert not bool(scratch.any())
    torch.cuda.synchronize()
    assert not bool(ws.any())


@pytest.mark.parametrize("which", ["q rows", "q utterances", "keys", "values", "groups of three", "groups of five"])
@pytest.mark.parametrize("kernel", [1, 2])
def test_strides_of_zero_and_odd_groups(which, kernel):
    B, R, S, Hkv, hd = 2, 40, 150, 2, 64
    G = {"groups of three": 3, "groups of five": 5}.get(which, 1)
    q, k, v = _rnd(1, B, R, Hkv * G, hd), _rnd(2, B, S, Hkv, hd), _rnd(3, B, S, Hkv, hd)
    if which == "q rows":
        q = q[:, :1].expand(B, R, Hkv, hd)
    elif which == "q utterances":
        q = q[:1].expand(B, R, Hkv, hd)
    elif which == "keys":
        k = k[:, :1].expand(B, S, Hkv, hd)
    elif which == "values":
        v = v[:, :, :1].expand(B, S, Hkv, hd)
    _lib.set_option("rows_kernel", kernel)
    try:
        out = asrq_b200.cross_attention(q, k, v)
    finally:
        _lib.set_option("rows_kernel", 0)
    check_rows(out, q, lambda b, r: (k[b], v[b]))
    asrq_b200.check_status()
