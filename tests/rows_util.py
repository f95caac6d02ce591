"""Attention over shared keys checked as a whole: every row of an utterance at once, each element by the worst case of the kernels' roundings and all of them
by what independent roundings come to, which a lost or doubled key of thousands does not pass."""
import math

import torch


def attend64(q, k, v, scale):
    """q (R, Hkv, G, hd), k and v (n, Hkv, hd), 64 bits: the result; the largest sum of a score's products' sizes per row; sum_t p_t^2 (v_t - result)^2."""
    q, k, v = (x.permute(*order).contiguous() for x, order in ((q, (1, 0, 2, 3)), (k, (1, 0, 2)), (v, (1, 0, 2))))
    Hkv, R, G, hd = q.shape
    rows = q.reshape(Hkv, R * G, hd)
    p = torch.softmax(rows @ k.transpose(1, 2) * scale, -1)
    size = (rows.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
    ref, p2 = p @ v, p * p
    spread = (p2 @ (v * v) - 2 * ref * (p2 @ v) + ref * ref * p2.sum(-1, keepdim=True)).clamp(min=0)
    shape = lambda x: x.view(Hkv, R, G, -1).permute(1, 0, 2, 3)  # noqa: E731
    return shape(ref), shape(size), shape(spread)


def check_utterance(got, q, k, v, scale=None):
    """got, q (R, heads, hd), k and v (n, key heads, hd) of one utterance.

    Each element: half a step of the result (eps / 2), the weights by half a step each (the quotient moves by at most eps |v|max), in fp16 also by 2^-36 of the largest for each of n; scores in 32
    bits, sums of hd products whose additions may cut instead of round, by hd 2^-22 of the products' sizes, and as much for the scaled difference,
    which moves the quotient by twice that of |v|max; 32-bit sums over n keys by n 2^-23 |v|max.
    All elements of many rows: a rounding to steps of at most eps |x| is off by eps |x| / sqrt(12) in the root mean square, the weights' roundings are independent and move the
    result by sum_t p_t d_t (v_t - result); scores and exponentials add less than 2^-22 of the products' sizes and 2^-18 to a weight's.  A quarter more for a finite sample."""
    R, Hq, hd = q.shape
    n, Hkv = k.shape[:2]
    assert tuple(got.shape) == tuple(q.shape) and got.dtype == q.dtype
    if n == 0:
        assert bool((got == 0).all())
        return
    scale, eps = hd ** -0.5 if scale is None else scale, torch.finfo(q.dtype).eps
    ref, size, spread = attend64(q.double().view(R, Hkv, -1, hd), k.double(), v.double(), scale)
    off = (got.double().view_as(ref) - ref).abs()
    vmax = v.double().abs().amax(0).amax(-1).view(1, Hkv, 1, 1)
    tol = eps / 2 * ref.abs() + vmax * (eps + (n * 2 ** -36 if q.dtype == torch.float16 else 0) + 4 * hd * 2 ** -22 * size + n * 2 ** -23) + 2 ** -24
    assert bool((off <= tol).all()), (n, float((off / tol).max()))
    weight = eps / math.sqrt(12) + 2 ** -22 * float(size.max()) + 2 ** -18
    bound = 1.25 * math.sqrt(eps ** 2 / 12 * float((ref * ref).mean()) + weight ** 2 * float(spread.mean())) + 2 ** -24
    rms = math.sqrt(float((off * off).mean()))
    assert rms <= bound, (n, rms, bound)
