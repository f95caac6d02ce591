"""What the rounding of the softmax weights may cost cross_attention and prefix_attention: an average of equal values is that value, and keys far
below the largest, but many, keep their part.  Scores are given: q = (1, 1, 0, ...), k = (a, b, 0, ...), scale ln 2, so that a key's weight is 2^(a + b) but for one unit in the last
place of the scale."""
import math

import pytest
import torch

import asrq_b200
from asrq_b200 import _lib

DEV = "cuda"
HEADS = 300  # more than the tensor-core kernel's blocks: most items are walked from end to end by one block, or one warp of the row kernel
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["row kernel", "tensor cores"])
def kernel(request):
    _lib.set_option("rows_kernel", 1 if request.param == "row kernel" else 2)
    yield
    _lib.set_option("rows_kernel", 0)
    asrq_b200.check_status()


def _queries(R, hd, dtype):
    q = torch.zeros(1, R, HEADS, hd, dtype=dtype, device=DEV)
    q[..., :2] = 1
    return q


def _keys(a, b, hd, dtype):
    """(1, n, HEADS, hd), the same for all heads: the exponents a + b."""
    k = torch.zeros(1, len(a), 1, hd, dtype=dtype, device=DEV)
    k[0, :, 0, 0], k[0, :, 0, 1] = a, b
    assert torch.equal(k[0, :, 0, 0].float(), a.float()) and torch.equal(k[0, :, 0, 1].float(), b.float())  # given exactly
    return k.expand(1, len(a), HEADS, hd)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("R,n,own", [(5, 4000, 0), (130, 4000, 0), (40, 700, 60)])
def test_average_of_equal_values(R, n, own, hd, dtype):
    """All keys have the same values: whatever the weights, and however they are rounded, the result is these values (in 32 bits to n 2^-23, here
    below half a step of either type: 4000 * 2^-23 = 4.8e-4 at the very most, a worst case of cut sums; the rounding to nearest then gives the value itself for sums that
    are off by less than 2^-12).  The later keys' weights lie just above a power of two, all on one side of what they are rounded to."""
    eps = torch.finfo(dtype).eps
    q, ln2 = _queries(R, hd, dtype), math.log(2.0)
    a = torch.full((n + own,), 3.0, device=DEV)
    b = torch.full((n + own,), math.log2(1 + 0.35 * eps), device=DEV).to(dtype).float()
    a[:96], b[:96] = 0, 0
    k = _keys(a, b, hd, dtype)
    value = torch.tensor([2 - eps, -1.0, 1 + eps, 0.0, 2 - eps, 3e-3, -2 + eps, 100.0] * (hd // 8), device=DEV).to(dtype)
    v = value.expand(1, n + own, 1, hd).contiguous().expand(1, n + own, HEADS, hd)
    if own:
        k1, v1 = (x[:, :n].transpose(1, 2) for x in (k, v))
        k2, v2 = (x[:, n:].transpose(1, 2).expand(R, HEADS, own, hd) for x in (k, v))
        out = asrq_b200.prefix_attention(q, k1, v1, k2, v2, torch.arange(R, device=DEV) % (own + 1), scale=ln2)
    else:
        out = asrq_b200.cross_attention(q, k, v, scale=ln2)
    assert torch.equal(out, value.expand_as(out))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R", [5, 130])
@pytest.mark.parametrize("low", [-20.25, -25.25, -28.0, -33.0])
def test_many_keys_far_below_one(low, R, dtype):
    """One key of weight 1 and value 0, n of weight 2^low and value 1: n 2^low / (1 + n 2^low).  Weights and result are rounded, by eps / 2 of themselves
    each; in fp16 a weight below 2^-25 of the largest by 2^-36 of that besides, scores in 32 bits by 34 * 2^-24, sums by n 2^-23 of themselves."""
    n, hd = 40000, 64
    eps = torch.finfo(dtype).eps
    a = torch.full((n + 1,), math.trunc(low), device=DEV, dtype=torch.float32)
    b = torch.full((n + 1,), low - math.trunc(low), device=DEV, dtype=torch.float32)
    a[700], b[700] = 0, 0
    v = torch.ones(1, n + 1, 1, hd, dtype=dtype, device=DEV)
    v[0, 700] = 0
    out = asrq_b200.cross_attention(_queries(R, hd, dtype), _keys(a, b, hd, dtype), v.expand(1, n + 1, HEADS, hd), scale=math.log(2.0)).double()
    mass = n * 2.0 ** low
    want = mass / (1 + mass)
    tol = want * (eps + 34 * 2 ** -24) + (n * 2 ** -36 if dtype == torch.float16 else 0) + want * n * 2 ** -23 + 2 ** -25
    assert bool(((out - want).abs() <= tol).all()), (want, float((out - want).abs().max()), tol)
