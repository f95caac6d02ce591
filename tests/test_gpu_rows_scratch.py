"""The scratch of cross_attention and prefix_attention: as much as the rows there are take, written within its bounds."""
import ctypes

import pytest
import torch

import asrq_b200
from asrq_b200 import _lib
from tests.beam_util import check_rows
from tests.gpu_util import CANARY, check_canary, lib_option, padded

DEV = "cuda"
pytestmark = pytest.mark.gpu


def _need(B, R, Hq, Hkv, hd, shared, own):
    return int(_lib.load().asrq_rows_attention_scratch_bytes(B, R, Hq, Hkv, hd, shared, own))


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [1, 5, 17, 64, 127, 128])
def test_no_more_than_its_rows_take(rows, hd):
    """A part is (rows, an odd number) x (hd values, maximum and sum) in 32 bits; an item has 64 parts and one of own keys at most."""
    with lib_option("rows_kernel", 2):
        for B, H, shared, own in ((2048, 20, 700, 40), (1, 2, 20000, 0), (1, 1, 45000, 30)):
            part, need = (rows | 1) * (hd + 2) * 4, _need(B, rows, H, H, hd, shared, own)
            assert need > 0 and need % part == 0 and need <= B * H * 65 * part, (B, H, need, part)
    with lib_option("rows_kernel", 2):  # one prompt of 2048 utterances, 17 beams: two parts an item
        assert _need(2048, rows, 20, 20, hd, 700, 40) <= 2048 * 20 * 2 * (rows + 1) * (hd + 2) * 4


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,R,Hq,Hkv,hd,P,M", [(2, 5, 4, 4, 64, 900, 0), (1, 17, 2, 2, 128, 3000, 33), (3, 3, 14, 2, 64, 500, 20), (1, 127, 2, 2, 64, 700, 9), (1, 300, 1, 1, 128, 2000, 11),
                                               (2, 1, 2, 2, 64, 5000, 7)])
def test_within_its_bounds(B, R, Hq, Hkv, hd, P, M, dtype):
    g = torch.Generator().manual_seed(R)
    rnd = lambda *shape: torch.randn(*shape, generator=g).to(dtype).to(DEV)  # noqa: E731
    q, k, v, k2, v2 = rnd(B, R, Hq, hd), rnd(B, Hkv, P, hd), rnd(B, Hkv, P, hd), rnd(B * R, Hkv, M, hd), rnd(B * R, Hkv, M, hd)
    n2 = torch.arange(B * R, device=DEV) % (M + 1)
    out, ws = padded((B, R, Hq, hd), dtype), torch.zeros(_lib.STATUS_BYTES, dtype=torch.uint8, device=DEV)
    s = asrq_b200.beam._strides
    with lib_option("rows_kernel", 2):
        need = _need(B, R, Hq, Hkv, hd, P, M)
        scratch = padded((need,), torch.uint8)
        scratch.fill_(0xFF)  # NaN: what is not written does not show
        _lib.call("asrq_prefix_attention", q.data_ptr(), s(q, 0, 1, 2), k.data_ptr(), s(k, 0, 1, 2), v.data_ptr(), s(v, 0, 1, 2), None, k2.data_ptr(), s(k2, 0, 1, 2),
                  v2.data_ptr(), s(v2, 0, 1, 2), n2.data_ptr(), B * R, out.data_ptr(), B, R, Hq, Hkv, hd, P, M, ctypes.c_float(hd ** -0.5),
                  _lib.F16 if dtype == torch.float16 else _lib.BF16, ws.data_ptr(), ws.numel(), scratch.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    n = n2.tolist()
    check_rows(out, q, lambda b, r: (torch.cat((k[b], k2[b * R + r, :, :n[b * R + r]]), 1).transpose(0, 1), torch.cat((v[b], v2[b * R + r, :, :n[b * R + r]]), 1).transpose(0, 1)))
    check_canary(out)
    check_canary(scratch)
    assert CANARY != 0xFF and not bool(ws.any())
    if 128 % (Hq // Hkv) == 0:  # (other groups run without it)
        assert need > 0 and bool((scratch != 0xFF).any())
    else:
        assert need == 0


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("own", [False, True])
def test_runs_where_there_is_no_memory_for_it(native, own, monkeypatch):
    """The allocator has nothing left but the output's memory: the kernels that need no scratch run."""
    K, H, hd, M = 128, 8, 128, 4
    B, P = (64, 700) if own else (4, 6000)
    g = torch.Generator().manual_seed(7)
    rnd = lambda *shape: torch.randn(*shape, generator=g).half().to(DEV)  # noqa: E731
    q, k, v, k2, v2, n2 = rnd(B, K, H, hd), rnd(B, H, P, hd), rnd(B, H, P, hd), rnd(B * K, H, M, hd), rnd(B * K, H, M, hd), torch.full((1,), M, device=DEV)
    if own:
        call = lambda: asrq_b200.prefix_attention(q, k, v, k2, v2, n2)  # noqa: E731
    else:
        call = lambda: asrq_b200.cross_attention(q, k.transpose(1, 2), v.transpose(1, 2))  # noqa: E731
    if not native:
        monkeypatch.setattr(asrq_b200.linear, "_native", None)
    with lib_option("rows_kernel", 2):
        want, need = call(), _need(B, K, H, H, hd, P, M if own else 0)
        assert need > (18 << 20)  # more than is left of the allocator's smallest large block, and of what the output's memory is rounded up to
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        block = torch.empty_like(want)  # the output's memory, in the allocator's hands when it is given back
        total = torch.cuda.get_device_properties(0).total_memory
        torch.cuda.set_per_process_memory_fraction(torch.cuda.memory_reserved() / total)
        try:
            with pytest.raises(torch.OutOfMemoryError):
                torch.empty(need, dtype=torch.uint8, device=DEV)
            del block
            got = call()
        finally:
            torch.cuda.set_per_process_memory_fraction(1.0)
    for out in (want, got):
        assert torch.equal(out, out) and bool(torch.isfinite(out).all())
    check_rows(got[:1, ::16].contiguous(), q[:1, ::16], lambda b, r: (torch.cat((k[b], k2[16 * r]), 1).transpose(0, 1), torch.cat((v[b], v2[16 * r]), 1).transpose(0, 1)) if own else
               (k[b].transpose(0, 1), v[b].transpose(0, 1)))
    check_rows(want[:1, ::16].contiguous(), q[:1, ::16], lambda b, r: (torch.cat((k[b], k2[16 * r]), 1).transpose(0, 1), torch.cat((v[b], v2[16 * r]), 1).transpose(0, 1)) if own else
               (k[b].transpose(0, 1), v[b].transpose(0, 1)))
