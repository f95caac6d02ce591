"""The engines' beam search when something about the engine or the call is not what it was: another output head, lengths of another shape, another default type."""
import warnings

import pytest
import torch

from asrq_b200 import qwen3 as Q
from asrq_b200 import whisper as W
from tests.gpu_util import DEV
from tests.qwen3_util import toy_models
from tests.whisper_util import load_fixture

transformers = pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu


def _whisper():
    cfg, sd, x, ids, logits, enc = load_fixture()
    m = W.WhisperForConditionalGenerationQ(transformers.WhisperConfig(**cfg))
    m.load_state_dict(sd)
    eng = W.WhisperEngine.from_model(m.half().to(DEV).eval())
    return eng, eng.encode(x)


def _qwen3():
    cfg, fm, q = toy_models()
    ids = torch.randint(0, cfg.vocab_size, (3, 9), generator=torch.Generator().manual_seed(1))
    return Q.Qwen3Engine.from_model(q.half().to(DEV)), fm.model.embed_tokens(ids).detach().half().to(DEV)


@pytest.mark.parametrize("use_graph", [False, True])
@pytest.mark.parametrize("make", [_whisper, _qwen3])
def test_another_output_head(make, use_graph):
    """Fewer tokens in the output head, then all of the embedding's again: the results are a new engine's with that head, and nothing is resized behind the
    caller's back."""
    eng, x = make()
    eng.beam_search(x, 5, 3, eos=7, use_graph=use_graph)
    full = eng.head
    assert full.shape[0] <= eng.embed.shape[0]
    for head in (full[:full.shape[0] - 24].contiguous(), full):
        eng.head = head
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            got = eng.beam_search(x, 5, 3, eos=7, use_graph=use_graph)
        other, y = make()
        other.head = head.clone()
        want = other.beam_search(y, 5, 3, eos=7, use_graph=use_graph)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("lengths", [torch.tensor([20]), torch.tensor([[20, 20]]), torch.tensor([20.0, 20.0]), [20, 20]])
def test_lengths_of_another_shape_or_type(lengths):
    eng, enc = _whisper()
    enc = enc[:2]
    with pytest.raises(ValueError, match="enc_lengths"):
        eng.beam_search(enc, 4, 3, enc_lengths=lengths)


@pytest.mark.parametrize("make", [_whisper, _qwen3])
def test_another_default_type(make):
    """A program that has set torch's default type to 16 bits gets the same search."""
    eng, x = make()
    want = eng.beam_search(x, 5, 3, eos=7)
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = eng.beam_search(x, 5, 3, eos=7)
    finally:
        torch.set_default_dtype(torch.float32)
    assert got[1].dtype == torch.float32 and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
