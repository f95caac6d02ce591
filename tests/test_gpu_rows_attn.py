"""cross_attention and prefix_attention against their definitions in 64 bits, on the GPU."""
import pytest
import torch

import asrq_b200
from asrq_b200 import _lib
from tests.beam_util import check_rows

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["row kernel", "tensor cores"])
def kernel(request):
    """Every test on both kernels, whatever the estimates would choose."""
    _lib.set_option("rows_kernel", 1 if request.param == "row kernel" else 2)
    yield
    _lib.set_option("rows_kernel", 0)
    asrq_b200.check_status()


def _rnd(seed, *shape, dtype=torch.float16, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,R,S,Hq,Hkv,hd", [
    (1, 1, 1, 1, 1, 64), (2, 1, 17, 2, 2, 128), (1, 5, 1500, 20, 20, 64), (3, 4, 31, 4, 1, 64), (2, 7, 33, 6, 2, 128), (1, 16, 100, 3, 3, 64),
    (2, 17, 65, 2, 2, 64), (1, 33, 200, 2, 1, 128), (1, 130, 129, 2, 2, 64), (9, 3, 257, 20, 20, 64), (1, 3, 4097, 1, 1, 128), (1, 2, 50, 21, 3, 64),
    (2, 200, 300, 4, 2, 128), (1, 448, 77, 1, 1, 64),
])
def test_cross(B, R, S, Hq, Hkv, hd, dtype):
    q, kv = _rnd(1, B, R, Hq, hd, dtype=dtype, std=1.5), _rnd(2, B, S, 2, Hkv, hd, dtype=dtype)
    k, v = kv[:, :, 0], kv[:, :, 1]
    check_rows(asrq_b200.cross_attention(q, k, v), q, lambda b, r: (k[b], v[b]))


@pytest.mark.parametrize("R", [1, 5, 40, 150])
@pytest.mark.parametrize("hd", [64, 128])
def test_cross_ragged(hd, R):
    """Lengths from nothing to all, some out of range; what lies past them is NaN and infinity."""
    B, S, H = 9, 200, 2
    lengths = torch.tensor([0, 1, 16, 31, 33, 199, 200, 5000, -3])
    q, k, v = _rnd(1, B, R, H, hd), _rnd(2, B, S, H, hd), _rnd(3, B, S, H, hd)
    for b, n in enumerate(lengths.clamp(0, S).tolist()):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    out = asrq_b200.cross_attention(q, k, v, lengths=lengths.to(DEV))
    n = lengths.clamp(0, S).tolist()
    check_rows(out, q, lambda b, r: (k[b, :n[b]], v[b, :n[b]]))


def test_cross_without_keys_and_without_rows():
    q, kv = _rnd(1, 2, 3, 4, 64), _rnd(2, 2, 0, 4, 64)
    assert not bool(asrq_b200.cross_attention(q, kv, kv).any())
    assert asrq_b200.cross_attention(q[:, :0], q, q).shape == (2, 0, 4, 64)
    assert asrq_b200.cross_attention(q[:0], q[:0], q[:0]).shape == (0, 3, 4, 64)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_cross_scale(scale):
    q, k, v = _rnd(1, 2, 5, 2, 64), _rnd(2, 2, 70, 2, 64), _rnd(3, 2, 70, 2, 64)
    check_rows(asrq_b200.cross_attention(q, k, v, scale=scale), q, lambda b, r: (k[b], v[b]), scale=scale)


def test_cross_layouts():
    """Head-major caches, a slice of a longer one, queries of a fused projection, a broadcast, and memory that is not aligned."""
    B, R, S, H, hd = 2, 6, 90, 3, 64
    cache = _rnd(2, 2, B, H, 128, hd)
    k, v = cache[0, :, :, 7:7 + S].transpose(1, 2), cache[1, :, :, 7:7 + S].transpose(1, 2)
    qkv = _rnd(1, B, R, 3, H, hd)
    q = qkv[:, :, 1]
    check_rows(asrq_b200.cross_attention(q, k, v), q, lambda b, r: (k[b], v[b]))
    k, v = k[:1].expand(B, S, H, hd), v[:1].expand(B, S, H, hd)
    check_rows(asrq_b200.cross_attention(q, k, v), q, lambda b, r: (k[b], v[b]))
    flat = _rnd(4, 3 + 2 * B * S * H * hd)
    k, v = flat[3:].view(2, B, S, H, hd)
    q = _rnd(5, 1 + B * R * H * hd)[1:].view(B, R, H, hd)
    check_rows(asrq_b200.cross_attention(q, k, v), q, lambda b, r: (k[b], v[b]))


@pytest.mark.parametrize("R", [3, 200])
def test_cross_of_peaked_and_extreme_scores(R):
    """One key far above the rest, equal keys, scores near the type's range."""
    q, k, v = _rnd(1, 3, R, 2, 64), _rnd(2, 3, 300, 2, 64), _rnd(3, 3, 300, 2, 64)
    k[0, 123] *= 30
    k[1] = k[1, :1]
    q[2] *= 100
    k[2] *= 30
    check_rows(asrq_b200.cross_attention(q, k, v), q, lambda b, r: (k[b], v[b]))


@pytest.mark.parametrize("R", [4, 200])
def test_cross_nan_reaches_its_row_only(R):
    q, k, v = _rnd(1, 2, R, 2, 64), _rnd(2, 2, 100, 2, 64), _rnd(3, 2, 100, 2, 64)
    want = asrq_b200.cross_attention(q, k, v)
    q[0, 2, 1, 5] = float("nan")
    got = asrq_b200.cross_attention(q, k, v)
    assert bool(torch.isnan(got[0, 2, 1]).all())
    got[0, 2, 1] = want[0, 2, 1]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,Hq,Hkv,hd,P,M,shared", [
    (1, 1, 1, 1, 64, 1, 1, 1), (1, 5, 16, 8, 128, 258, 40, 33), (2, 3, 4, 2, 64, 50, 9, 0), (3, 16, 2, 1, 128, 100, 20, 0), (1, 33, 3, 1, 64, 70, 5, 0),
    (2, 8, 12, 4, 128, 17, 300, 0), (1, 64, 2, 1, 128, 1000, 60, 0), (1, 70, 4, 2, 64, 500, 10, 7), (20, 2, 8, 8, 64, 33, 33, 0), (1, 5, 8, 2, 128, 5000, 16, 16),
    (1, 200, 2, 2, 64, 300, 3, 0),
])
def test_prefix(B, K, Hq, Hkv, hd, P, M, shared, dtype):
    q = _rnd(1, B, K, Hq, hd, dtype=dtype, std=1.5)
    kp, vp = _rnd(2, 2, B, Hkv, P, hd, dtype=dtype)
    ks, vs = _rnd(3, 2, B * K, Hkv, M, hd, dtype=dtype)
    mine = torch.tensor([shared]) if shared else torch.randint(0, M + 1, (B * K,), generator=torch.Generator().manual_seed(5))
    n = mine.tolist() * (B * K if shared else 1)
    out = asrq_b200.prefix_attention(q, kp, vp, ks, vs, mine.to(DEV))

    def keys(b, r):
        i = b * K + r
        return torch.cat([kp[b], ks[i, :, :n[i]]], 1).transpose(0, 1), torch.cat([vp[b], vs[i, :, :n[i]]], 1).transpose(0, 1)

    check_rows(out, q, keys)


@pytest.mark.parametrize("K", [4, 90])
@pytest.mark.parametrize("hd", [64, 128])
def test_prefix_ragged(hd, K):
    """Prompts and beams of every kind of length, nothing among them; NaN and infinity behind each length, and in one beam's own values: no other
    beam is any different for it."""
    B, H, P, M = 4, 2, 60, 40
    np_ = torch.tensor([0, 1, 60, 33])
    ns = torch.randint(0, M + 1, (B * K,), generator=torch.Generator().manual_seed(2))
    ns[0], ns[1], ns[K] = 0, M, 0
    q, (kp, vp), (ks, vs) = _rnd(1, B, K, 2 * H, hd), _rnd(2, 2, B, H, P, hd), _rnd(3, 2, B * K, H, M, hd)
    for b in range(B):
        kp[b, :, np_[b]:], vp[b, :, np_[b]:] = float("inf"), float("nan")
    for i in range(B * K):
        ks[i, :, ns[i]:], vs[i, :, ns[i]:] = float("nan"), float("inf")
    out = asrq_b200.prefix_attention(q, kp, vp, ks, vs, ns.to(DEV), prefix_lengths=np_.to(DEV))

    def keys(b, r):
        i = b * K + r
        return (torch.cat([kp[b, :, :np_[b]], ks[i, :, :ns[i]]], 1).transpose(0, 1), torch.cat([vp[b, :, :np_[b]], vs[i, :, :ns[i]]], 1).transpose(0, 1))

    check_rows(out, q, keys)
    i = 2 * K + 1
    ns[i] = 7
    out = asrq_b200.prefix_attention(q, kp, vp, ks, vs, ns.to(DEV), prefix_lengths=np_.to(DEV))
    ks[i, :, 3], vs[i, :, 5] = float("inf"), float("-inf")
    got = asrq_b200.prefix_attention(q, kp, vp, ks, vs, ns.to(DEV), prefix_lengths=np_.to(DEV))
    assert not bool(torch.isfinite(got[2, 1]).all())
    got[2, 1] = out[2, 1]
    assert torch.equal(got, out)


def test_prefix_without_either_part():
    q, some, none = _rnd(1, 2, 3, 4, 64), _rnd(2, 2, 2, 10, 64), _rnd(2, 2, 2, 0, 64)
    own, no_own = _rnd(3, 6, 2, 5, 64), _rnd(3, 6, 2, 0, 64)
    n = torch.tensor([5], device=DEV)
    check_rows(asrq_b200.prefix_attention(q, some, some, no_own, no_own, n), q, lambda b, r: (some[b].transpose(0, 1),) * 2)
    check_rows(asrq_b200.prefix_attention(q, none, none, own, own, n), q, lambda b, r: (own[b * 3 + r].transpose(0, 1),) * 2)
    assert not bool(asrq_b200.prefix_attention(q, none, none, no_own, no_own, n).any())


def test_prefix_views_of_longer_caches():
    """The prompt's part of the caches that prefill wrote, and one layer of the beams' own."""
    B, K, Hq, Hkv, hd, P, M = 2, 5, 4, 2, 128, 37, 20
    cache, own = _rnd(1, 2, B, Hkv, 80, hd), _rnd(2, 3, 2, B * K, Hkv, M, hd)
    q = _rnd(3, B, K, (Hq + 2 * Hkv) * hd)[..., :Hq * hd].view(B, K, Hq, hd)
    kp, vp, (ks, vs) = cache[0, :, :, :P], cache[1, :, :, :P], own[1]
    n = torch.tensor([11], device=DEV)
    check_rows(asrq_b200.prefix_attention(q, kp, vp, ks, vs, n), q,
               lambda b, r: (torch.cat([kp[b], ks[b * K + r, :, :11]], 1).transpose(0, 1), torch.cat([vp[b], vs[b * K + r, :, :11]], 1).transpose(0, 1)))


def test_offsets_past_32_bits():
    """A prompt of 2.2e9 values of which the last utterance's last positions decide."""
    P, H = 140000, 62
    kp = torch.zeros(2, H, P, 128, dtype=torch.float16, device=DEV)
    kp[1, -1, -40:] = _rnd(2, 40, 128)
    q, own = _rnd(1, 2, 3, H, 128), _rnd(3, 6, H, 4, 128)
    n = torch.tensor([4], device=DEV)
    out = asrq_b200.prefix_attention(q, kp, kp, own, own, n)
    k, v = (torch.cat([kp[1, -1:], own[5, -1:, :4]], 1).transpose(0, 1),) * 2
    check_rows(out[1:, 2:, -1:].contiguous(), q[1:, 2:, -1:], lambda b, r: (k, v))


def test_captured_with_lengths_on_the_device():
    """A graph is replayed as lengths and inputs change; two graphs of one stream replayed on two streams at once do not meet."""
    B, K, H, hd, P, M = 2, 5, 4, 64, 600, 30
    q, (kp, vp), (ks, vs) = _rnd(1, B, K, H, hd), _rnd(2, 2, B, H, P, hd), _rnd(3, 2, B * K, H, M, hd)
    big = _rnd(4, B, 150, H, hd)
    n, p = torch.tensor([3], device=DEV), torch.tensor([P, 100], device=DEV)

    def calls():
        return (asrq_b200.prefix_attention(q, kp, vp, ks, vs, n, prefix_lengths=p), asrq_b200.cross_attention(q, kp.transpose(1, 2), vp.transpose(1, 2), lengths=p),
                asrq_b200.cross_attention(big, kp.transpose(1, 2), vp.transpose(1, 2), lengths=p))

    calls()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(calls())
        graphs.append(g)
    for own, first in ((1, 600), (30, 0), (0, 17)):
        n.fill_(own)
        p[0] = first
        want = calls()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
