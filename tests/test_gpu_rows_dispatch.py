"""cross_attention and prefix_attention as large calls divide them: blocks that take one unit after another, items with and without parts in one
call, units without keys between others; and the choice between the kernels as it is made when nothing forces it.  All rows against 64 bits."""
import pytest
import torch

import asrq_b200
from asrq_b200 import _lib
from tests.gpu_util import lib_option
from tests.rows_util import check_utterance

DEV = "cuda"
TYPES = [torch.float16, torch.bfloat16]
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def status():
    yield
    asrq_b200.check_status()


def _rnd(seed, *shape, dtype=torch.float16, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * std).to(dtype)


def _parts(B, R, Hq, Hkv, hd, shared, own):
    """How many parts the call leaves for a join, and its items (utterance, key head, 128 rows)."""
    rows = R * (Hq // Hkv)
    need = int(_lib.load().asrq_rows_attention_scratch_bytes(B, R, Hq, Hkv, hd, shared, own))
    return need // ((min(rows, 128) | 1) * (hd + 2) * 4), B * Hkv * -(-rows // 128)


def _cross(B, R, Hq, Hkv, hd, S, dtype, lengths=None):
    q, kv = _rnd(1, B, R, Hq, hd, dtype=dtype, std=1.5), _rnd(2, B, S, 2, Hkv, hd, dtype=dtype)
    k, v = kv[:, :, 0], kv[:, :, 1]
    if lengths is not None:
        for b, n in enumerate(lengths):
            k[b, n:], v[b, n:] = float("nan"), float("inf")
        out = asrq_b200.cross_attention(q, k, v, lengths=torch.tensor(lengths, device=DEV))
    else:
        out = asrq_b200.cross_attention(q, k, v)
    for b in range(B):
        n = S if lengths is None else lengths[b]
        check_utterance(out[b], q[b], k[b, :n], v[b, :n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,R,H,hd,S", [(16, 224, 20, 64, 700), (13, 300, 8, 128, 500), (8, 128, 40, 64, 260), (5, 129, 31, 128, 1000)])
def test_more_items_than_blocks(B, R, H, hd, S, dtype):
    """Whole items, several to a block, and behind them items that are divided where there are keys enough."""
    slots = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    with lib_option("rows_kernel", 2):
        parts, items = _parts(B, R, H, H, hd, S, 0)
        assert items > slots and (parts > 0) == (S >= 4 * (96 if hd == 64 else 64))  # fewer than four tiles of keys are not divided
        _cross(B, R, H, H, hd, S, dtype)
    assert _parts(16, 224, 20, 20, 64, 1500, 0)[0] > 0  # and so does a prompt's cross-attention by itself


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,R,H,hd,S", [(20, 200, 20, 64, 420), (24, 130, 10, 128, 300)])
def test_units_without_keys_between_others(B, R, H, hd, S, dtype):
    lengths = [0 if b % 3 == 1 else (S if b % 4 == 0 else 1 + (b * 97) % S) for b in range(B)]
    lengths[0], lengths[-1] = 0, S - 1
    with lib_option("rows_kernel", 2):
        _cross(B, R, H, H, hd, S, dtype, lengths)
        _cross(B, R, H, H, hd, S, dtype, [0] * (B - 1) + [S])
        _cross(B, R, H, H, hd, S, dtype, [S] + [0] * (B - 1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,K,Hq,Hkv,hd,P,M", [(40, 9, 16, 8, 64, 300, 20), (41, 33, 16, 8, 128, 200, 30), (3, 150, 8, 4, 64, 2500, 17)])
def test_own_keys_behind_more_items_than_blocks(B, K, Hq, Hkv, hd, P, M, dtype):
    q, (kp, vp), (ks, vs) = _rnd(1, B, K, Hq, hd, dtype=dtype, std=1.5), _rnd(2, 2, B, Hkv, P, hd, dtype=dtype), _rnd(3, 2, B * K, Hkv, M, hd, dtype=dtype)
    np_, ns = [(b * 53) % (P + 1) for b in range(B)], [(i * 7) % (M + 1) for i in range(B * K)]
    np_[0], np_[-1], ns[0], ns[1] = P, 0, 0, M
    for b in range(B):
        kp[b, :, np_[b]:], vp[b, :, np_[b]:] = float("nan"), float("inf")
    with lib_option("rows_kernel", 2):
        assert _parts(B, K, Hq, Hkv, hd, P, M)[0] > 0
        out = asrq_b200.prefix_attention(q, kp, vp, ks, vs, torch.tensor(ns, device=DEV), prefix_lengths=torch.tensor(np_, device=DEV))
    for b in range(B):
        for j in range(0, K, 1 if K < 10 else 7):
            i = b * K + j
            check_one = (torch.cat([kp[b, :, :np_[b]], ks[i, :, :ns[i]]], 1).transpose(0, 1), torch.cat([vp[b, :, :np_[b]], vs[i, :, :ns[i]]], 1).transpose(0, 1))
            check_utterance(out[b, j:j + 1], q[b, j:j + 1], *check_one)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kernel", [0, 1, 2])
@pytest.mark.parametrize("B,R,Hq,Hkv,hd,S", [
    (1, 5, 20, 20, 64, 1500), (16, 5, 20, 20, 64, 1500), (16, 16, 20, 20, 64, 1500), (16, 17, 20, 20, 64, 1500), (4, 32, 20, 20, 64, 1500), (1, 64, 20, 20, 64, 1500),
    (2, 64, 16, 8, 128, 1500), (16, 20, 8, 8, 128, 700), (2, 40, 12, 4, 64, 900), (3, 448, 20, 20, 64, 1500), (1, 300, 8, 1, 128, 4097), (2, 20, 4, 4, 64, 63), (2, 20, 4, 4, 64, 64),
])
def test_either_side_of_the_choice(B, R, Hq, Hkv, hd, S, kernel, dtype):
    """The shapes around which the choice changes, by the choice and by either kernel."""
    with lib_option("rows_kernel", kernel):
        _cross(B, R, Hq, Hkv, hd, S, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [45000, 300000])
@pytest.mark.parametrize("kernel", [1, 2])
def test_long_keys_to_the_last(n, kernel, dtype):
    """The sum of all roundings over a long axis in few and in many parts stays that of independent roundings."""
    with lib_option("rows_kernel", kernel):
        _cross(1, 33, 2, 2, 64, n, dtype)
