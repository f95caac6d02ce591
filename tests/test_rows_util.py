"""The check of attention over shared keys finds what it is there to find: mistakes planted in a 64-bit result (no GPU)."""
import pytest
import torch

from tests.rows_util import attend64, check_utterance


def _case(dtype, R, n, H, hd):
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(m, H, hd, generator=g) for m in (R, n, n))
    return (q * 1.5).to(dtype), k.to(dtype), v.to(dtype)


def _result(q, k, v, keep):
    """As a kernel would return it: weights and result rounded, the sum that of the rounded weights."""
    q64, k64, v64 = q.double(), k[keep].double(), v[keep].double()
    s = torch.einsum("rhd,nhd->rhn", q64, k64) * q.shape[-1] ** -0.5
    w = (s - s.amax(-1, keepdim=True)).exp().to(q.dtype).double()
    return (torch.einsum("rhn,nhd->rhd", w, v64) / w.sum(-1, keepdim=True)).to(q.dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,n,H,hd", [(40, 4097, 1, 128), (224, 700, 2, 64), (64, 1500, 2, 64)])
def test_a_lost_or_doubled_key_shows(R, n, H, hd, dtype):
    q, k, v = _case(dtype, R, n, H, hd)
    every = torch.arange(n)
    check_utterance(_result(q, k, v, every), q, k, v)
    for keep in (every[every != 77], every[:n - 1], every[(every < 320) | (every >= 352)], torch.cat([every, every[5:6]])):
        with pytest.raises(AssertionError):
            check_utterance(_result(q, k, v, keep), q, k, v)


def test_the_reference_is_the_definition():
    q, k, v = (x.double() for x in _case(torch.float16, 6, 50, 2, 64))
    ref, size, spread = attend64(q.view(6, 1, 2, 64), k[:, :1], v[:, :1], 0.2)
    for r in range(6):
        for g in range(2):
            p = torch.softmax(k[:, 0] @ q[r, g] * 0.2, 0)
            out = p @ v[:, 0]
            assert torch.allclose(ref[r, 0, g], out, rtol=1e-12, atol=1e-14)
            assert torch.allclose(spread[r, 0, g], (p * p) @ (v[:, 0] - out) ** 2, rtol=1e-9, atol=1e-14)
            assert abs(float(size[r, 0, g, 0]) - float((k[:, 0].abs() @ q[r, g].abs()).max() * 0.2)) < 1e-9
