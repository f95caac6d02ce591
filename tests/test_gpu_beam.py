"""beam_select and beam_reorder against their definitions, on the GPU."""
import pytest
import torch

import asrq_b200
from tests.beam_util import check_select

DEV = "cuda"
pytestmark = pytest.mark.gpu


def _logits(B, K, V, dtype, seed, offset=0, pad=0):
    """(B, K, V) logits that start ``offset`` values into their memory and whose rows lie ``pad`` values apart."""
    g = torch.Generator().manual_seed(seed)
    flat = torch.full((offset + B * K * (V + pad),), float("nan"), dtype=dtype)
    x = flat[offset:].view(B, K, V + pad)[:, :, :V]
    x.copy_((torch.randn(B, K, V, generator=g) * 3).to(dtype))
    flat = flat.to(DEV)
    return flat[offset:].view(B, K, V + pad)[:, :, :V]


def _scores(B, K, seed):
    return (-torch.rand(B, K, generator=torch.Generator().manual_seed(seed + 1)).cumsum(1) * 4).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n,offset,pad", [
    (1, 1, 1, 1, 0, 0), (1, 1, 7, 7, 1, 0), (2, 3, 9, 5, 3, 1), (1, 5, 51866, 5, 0, 0), (3, 5, 1000, 10, 0, 24), (10, 2, 333, 4, 5, 0),
    (1, 32, 257, 32, 0, 0), (12, 7, 2049, 14, 2, 7), (1, 3, 151936, 6, 0, 0), (11, 1, 65537, 32, 1, 2), (150, 4, 63, 4, 0, 0), (1, 4, 8, 32, 0, 0),
])
def test_select(B, K, V, n, offset, pad, dtype):
    logits, scores = _logits(B, K, V, dtype, B * 7 + V, offset, pad), _scores(B, K, V)
    check_select(asrq_b200.beam_select(logits, scores, n), logits, scores, n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_select_at_the_limits(dtype):
    V = 65536 * 4
    logits, scores = _logits(1, 32, V, dtype, 5), _scores(1, 32, 5)
    check_select(asrq_b200.beam_select(logits, scores, 32), logits, scores, 32)
    V = 65536 * 128  # one beam: 128 segments
    logits, scores = _logits(1, 1, V, dtype, 6), _scores(1, 1, 6)
    check_select(asrq_b200.beam_select(logits, scores, 8), logits, scores, 8)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("what", ["all equal", "few values", "zeros of both signs", "equal beams", "mostly hidden", "all but three hidden", "ascending", "large"])
def test_select_ties_and_hidden_tokens(what, dtype):
    B, K, V, n = 3, 4, 6001, 16
    logits, scores = _logits(B, K, V, dtype, 3), _scores(B, K, 3)
    g = torch.Generator().manual_seed(9)
    if what == "all equal":
        logits.fill_(1.5)
        scores.fill_(-2.0)
    elif what == "few values":
        logits.copy_(torch.randint(-2, 2, (B, K, V), generator=g))
    elif what == "zeros of both signs":
        logits.copy_(torch.where(torch.rand(B, K, V, generator=g) < 0.5, 0.0, -0.0))
    elif what == "equal beams":  # at different alignments: the rows are 6001 values apart
        logits.copy_(logits[:, :1].clone().expand(B, K, V))
        scores.fill_(-1.25)
    elif what == "mostly hidden":
        logits.masked_fill_((torch.rand(B, K, V, generator=g) < 0.999).to(DEV), float("-inf"))
    elif what == "all but three hidden":
        keep = logits[:, :, [5, 77, 6000]].clone()
        logits.fill_(float("-inf"))
        logits[:, :, [5, 77, 6000]] = keep
    elif what == "ascending":
        logits.copy_((torch.arange(V) // 8 - 400).expand(B, K, V).clamp(-300, 300))
    else:
        logits.mul_(0).add_(torch.finfo(dtype).max)
        logits[:, :, ::3] = torch.finfo(dtype).min
    check_select(asrq_b200.beam_select(logits, scores, n), logits, scores, n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_select_without_hypothesis(dtype):
    """Scores of -inf (the first step), +inf and NaN, rows of NaN, +inf and of nothing: offered at -inf, lowest first."""
    B, K, V, n = 4, 5, 700, 10
    logits, scores = _logits(B, K, V, dtype, 8), _scores(B, K, 8)
    scores[0, 1:] = float("-inf")
    scores[1, 0], scores[1, 1], scores[1, 2] = float("nan"), float("inf"), float("-inf")
    logits[2, 0, 3], logits[2, 1, 699], logits[2, 2] = float("nan"), float("inf"), float("-inf")
    logits[3] = float("-inf")
    logits[3, 4, 650] = 2.0
    check_select(asrq_b200.beam_select(logits, scores, n), logits, scores, n)
    scores.fill_(float("-inf"))
    check_select(asrq_b200.beam_select(logits, scores, n), logits, scores, n)


@pytest.mark.parametrize("eos", [0, 3, 699])
def test_select_with_ended_beams(eos):
    B, K, V, n = 4, 5, 700, 10
    logits, scores = _logits(B, K, V, torch.float16, 8), _scores(B, K, 8)
    finished = torch.zeros(B, K, dtype=torch.bool, device=DEV)
    finished[1, 2] = True
    finished[2, :4] = True
    finished[3] = True
    logits[1, 2] = float("nan")  # not looked at
    scores[2, 1] = float("-inf")
    logits[0, 0, eos] = 20.0
    check_select(asrq_b200.beam_select(logits, scores, n, finished=finished, eos=eos), logits, scores, n, finished, eos)


def test_select_twice_at_once_and_captured():
    """Two streams at once, and a graph replayed with other inputs: the calls share nothing."""
    sets = [(_logits(4, 5, 51866, torch.float16, s), _scores(4, 5, s)) for s in range(4)]
    alone = [asrq_b200.beam_select(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(asrq_b200.beam_select(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, alone[i % 4]))
    logits, scores = sets[0][0].clone(), sets[0][1].clone()
    asrq_b200.beam_select(logits, scores)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = asrq_b200.beam_select(logits, scores)
    for (x, s), want in zip(sets, alone):
        logits.copy_(x)
        scores.copy_(s)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def _reordered(cache, parents, length):
    B, K = parents.shape
    out = cache.clone()
    for b in range(B):
        for k in range(K):
            p = int(parents[b, k])
            if 0 <= p < K and length > 0:
                out[:, b * K + k, :, :length] = cache[:, b * K + p, :, :length]
    return out


@pytest.mark.parametrize("L,B,K,H,M,hd,length,dtype", [
    (4, 1, 5, 3, 33, 64, 20, torch.float16), (2, 3, 8, 2, 17, 128, 17, torch.bfloat16), (3, 2, 9, 1, 300, 8, 299, torch.float16),
    (2, 1, 32, 2, 5, 64, 3, torch.float16), (2, 2, 16, 2, 5, 4, 1, torch.float32), (2, 2, 2, 1, 9, 64, 0, torch.float16), (1, 7, 1, 2, 9, 64, 5, torch.float16),
    (2, 2, 3, 2, 9, 64, 50, torch.float16), (2, 2, 3, 2, 9, 64, -4, torch.float16),
])
@pytest.mark.parametrize("on_device", [False, True])
def test_reorder(L, B, K, H, M, hd, length, dtype, on_device):
    g = torch.Generator().manual_seed(L * 100 + K)
    cache = torch.randn(L, B * K, H, M, hd, generator=g).to(dtype).to(DEV)
    cache[0, 0, 0, 0, :4] = torch.tensor([float("nan"), float("inf"), -0.0, 1.0])
    parents = torch.randint(0, K, (B, K), generator=g).to(DEV)
    want = _reordered(cache, parents, min(max(length, 0), M))
    got = asrq_b200.beam_reorder(cache, parents, torch.tensor([length], device=DEV) if on_device else length)
    assert got.data_ptr() == cache.data_ptr()
    as_int = {2: torch.int16, 4: torch.int32}[cache.element_size()]
    assert torch.equal(cache.view(as_int), want.view(as_int))


def test_reorder_of_all_one_parent_a_cycle_and_none():
    K = 6
    base = torch.randn(2, 3 * K, 2, 40, 64, device=DEV).half()
    parents = torch.tensor([[2] * K, [1, 2, 3, 4, 5, 0], list(range(K))], device=DEV)
    want = _reordered(base, parents, 31)
    assert torch.equal(asrq_b200.beam_reorder(base.clone(), parents, 31), want)
    parents[0, 1], parents[1, 3] = -1, K  # no beams: these rows stay
    want = _reordered(base, parents, 31)
    assert torch.equal(asrq_b200.beam_reorder(base.clone(), parents, 31), want)


def test_reorder_of_a_cache_past_32_bits():
    """2.2e9 values: offsets that do not fit 32 bits."""
    K, M, H = 2, 4200, 32
    cache = torch.zeros(64, 2 * K, H, M, 64, dtype=torch.float16, device=DEV)
    cache[-1, -2:, -1, -5:] = torch.randn(2, 5, 64, device=DEV).half()
    old = cache[-1, -2:].clone()
    asrq_b200.beam_reorder(cache, torch.tensor([[0, 1], [1, 0]], device=DEV), M)
    assert torch.equal(cache[-1, -2:], old.flip(0)) and not bool(cache[0].any())
