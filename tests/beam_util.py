"""The operators of decoding with beams in 64 bits, from their definitions, and the bounds that their kernels' roundings give."""
import math

import torch


def select64(logits, scores, n, finished=None, eos=None):
    """(values, places): the n largest of every utterance, of equal ones the lowest k * V + v, in 64 bits on the CPU."""
    B, K, V = logits.shape
    values, places = [], []
    for b in range(B):
        table = torch.full((K, V), float("-inf"), dtype=torch.float64)
        for k in range(K):
            s = float(scores[b, k])
            if not math.isfinite(s):
                continue
            if finished is not None and bool(finished[b, k]):
                table[k, eos] = s
                continue
            x = logits[b, k].double().cpu()
            if not math.isfinite(float(x.max())) or bool(torch.isnan(x).any()):
                continue
            table[k] = s + (x - torch.logsumexp(x, 0))
        order = torch.sort(table.view(-1), descending=True, stable=True)
        values.append(order.values[:min(n + 1, K * V)])
        places.append(order.indices[:n])
    return values, torch.stack(places)


def check_select(got, logits, scores, n, finished=None, eos=None):
    """The kernel's sums are in 32 bits: exponentials off by 2^-22 and by 2^-24 for each unit that the logit lies below the maximum (weighted: at most ln V + 1, below 14), partial sums of 16 and the
    joining of them by 20 * 2^-24, so the normalisation by less than 4e-6; the result is rounded to 32 bits.  Where two candidates are not equal, but nearer than
    twice that, either may come first."""
    B, K, V = logits.shape
    values, places = select64(logits, scores, n, finished, eos)
    out, parents, tokens = (t.cpu() for t in got[:3])
    assert out.dtype == torch.float32 and parents.dtype == tokens.dtype == torch.int64 and tuple(out.shape) == tuple(parents.shape) == tuple(tokens.shape) == (B, n)
    for b in range(B):
        ref = values[b]
        for i in range(n):
            r, o = float(ref[i]), float(out[b, i])
            assert (r == o) if math.isinf(r) else abs(r - o) <= 4e-6 + 2 ** -24 * abs(r), (b, i, r, o)
            near = [j for j in (i - 1, i + 1) if 0 <= j < len(ref) and not math.isinf(r) and 0 < abs(float(ref[j]) - r) < 8e-6]
            if not near:
                assert int(parents[b, i]) * V + int(tokens[b, i]) == int(places[b, i]), (b, i, int(parents[b, i]), int(tokens[b, i]), int(places[b, i]))
    flat = parents * V + tokens
    assert all(len(set(row.tolist())) == n for row in flat)
    if finished is not None:
        over = got[3].cpu()
        assert over.dtype == torch.bool and torch.equal(over, finished.cpu().gather(1, parents) | (tokens == eos))


def _rows64(q, k, v, scale):
    """q (rows, Hkv, G, hd), k and v (n, Hkv, hd) in 64 bits -> the result and what its tolerance goes by."""
    s = torch.einsum("rhgd,nhd->rhgn", q, k) * scale
    size = torch.einsum("rhgd,nhd->rhgn", q.abs(), k.abs()).amax(-1, keepdim=True) * abs(scale)
    return torch.einsum("rhgn,nhd->rhgd", torch.softmax(s, -1), v), size, v.abs().amax(0).amax(-1).view(1, -1, 1, 1)


def check_rows(got, q, keys_of, scale=None):
    """``keys_of(b, r)``: keys and values (n, Hkv, hd) of row r of utterance b.  Against 64 bits, with the bound of the kernels' roundings: the result by half a step (eps / 2); the weights by half a step each, which moves the
    quotient by at most eps / 2 (|v| + |out|) <= eps |v|max, in fp16 also by 2^-25 for each of n weights that have left the normal range; the scores, sums of hd products in 32 bits whose additions
    may cut instead of round, by hd 2^-22 of the sum of the products' sizes, and as much again for the scaled difference, which moves a weight by
    as much relative to itself and the quotient by twice that of |v|max; 32-bit sums over n keys by n 2^-23 |v|max."""
    B, R, Hq, hd = q.shape
    scale = hd ** -0.5 if scale is None else scale
    eps = torch.finfo(q.dtype).eps
    assert tuple(got.shape) == tuple(q.shape) and got.dtype == q.dtype and got.is_contiguous()
    for b in range(B):
        for r in range(R):
            k, v = keys_of(b, r)
            n = k.shape[0]
            mine = got[b, r].double()
            if n == 0:
                assert bool((mine == 0).all()), (b, r)
                continue
            ref, size, vmax = _rows64(q[b, r].double().view(1, k.shape[1], -1, hd), k.double(), v.double(), scale)
            tol = eps / 2 * ref.abs() + vmax * (eps + (n * 2 ** -25 if q.dtype == torch.float16 else 0) + 4 * hd * 2 ** -22 * size + n * 2 ** -23) + 2 ** -24
            off = (mine.view_as(ref) - ref).abs()
            assert bool((off <= tol).all()), (b, r, n, float((off / tol).max()))
