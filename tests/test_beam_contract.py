"""What the C entry points of the operators of decoding with beams refuse before they launch anything: memory their vector stores cannot take (no GPU needed)."""
import ctypes

import pytest

from asrq_b200 import _lib

I3 = ctypes.c_int64 * 3
S = I3(64, 64, 64)


def _buffer():
    buf = ctypes.create_string_buffer(1024 + 16)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def _cross(p, out, ws, scratch):
    return _lib.load().asrq_cross_attention(p, S, p, S, p, S, None, out, 1, 1, 2, 2, 64, 4, 1.0, 0, ws, 256, scratch, 64, None)


def _prefix(p, out, ws, scratch):
    return _lib.load().asrq_prefix_attention(p, S, p, S, p, S, None, p, S, p, S, p, 1, out, 1, 2, 2, 2, 64, 4, 4, 1.0, 0, ws, 256, scratch, 64, None)


@pytest.mark.parametrize("call", [_cross, _prefix])
@pytest.mark.parametrize("which", ["out", "ws", "scratch"])
@pytest.mark.parametrize("off", [2, 4, 8])
def test_attention_refuses_memory_that_is_not_aligned(call, which, off):
    keep, p = _buffer()
    at = dict(out=p, ws=p, scratch=p)
    at[which] += off
    assert call(p, **at) == -3 and "16-byte aligned" in _lib.last_error()


def test_reorder_refuses_a_workspace_that_is_not_aligned():
    keep, p = _buffer()
    assert _lib.load().asrq_beam_reorder(p, p, None, 2, 1, 1, 2, 1, 4, 16, p + 4, 256, None) == -3
    assert "16-byte aligned" in _lib.last_error()
