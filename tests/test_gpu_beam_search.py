"""Beam search of the two engines: every step's selection against its definition, and every hypothesis' logits against the same tokens run through the
greedy engine, which shares neither caches nor attention kernels with it."""
import pytest
import torch

import asrq_b200
from asrq_b200 import beam as BM
from asrq_b200 import qwen3 as Q
from asrq_b200 import whisper as W
from tests.beam_util import check_select
from tests.gpu_util import DEV
from tests.qwen3_util import toy_models
from tests.whisper_util import load_fixture

transformers = pytest.importorskip("transformers")
pytestmark = pytest.mark.gpu


class _Seen:
    """Every call of beam_select with what it returned."""

    def __init__(self, monkeypatch):
        self.calls = []
        inner = BM.beam_select

        def select(logits, scores, n=None, finished=None, eos=None):
            out = inner(logits, scores, n, finished=finished, eos=eos)
            keep = lambda t: None if t is None else t.clone()  # noqa: E731
            self.calls.append((logits.clone(), scores.clone(), out[0].shape[1], keep(finished), eos, tuple(t.clone() for t in out)))
            return out

        monkeypatch.setattr(BM, "beam_select", select)

    def check(self):
        for logits, scores, n, finished, eos, out in self.calls:
            check_select(out, logits, scores, n, finished, eos)

    def hypotheses(self):
        """After each call the hypotheses as token lists [utterance][beam]."""
        found, now = [], None
        for *_, out in self.calls:
            parents, tokens = out[1].tolist(), out[2].tolist()
            now = [[(now[b][p] if now else []) + [t] for p, t in zip(pb, tb)] for b, (pb, tb) in enumerate(zip(parents, tokens))]
            found.append(now)
        return found


def _check_search(seen, ids, scores, eos, length_penalty, rescored):
    """``rescored(b, tokens)``: the logits (len(tokens), V) that those tokens were chosen from, by another path.  The logits of two 16-bit paths through the same
    layers are held to 1e-2 of the largest, as elsewhere."""
    seen.check()
    hyps = seen.hypotheses()
    B, K, steps = ids.shape
    last, out = hyps[-1], seen.calls[-1][-1]
    for b in range(B):
        ranked = []
        for k in range(K):
            tokens = last[b][k]
            n = tokens.index(eos) + 1 if eos is not None and eos in tokens else steps
            ranked.append((float(out[0][b, k]) / n ** length_penalty, k))
        order = [k for _, k in sorted(ranked, key=lambda x: (-x[0], x[1]))]
        assert ids[b].tolist() == [last[b][k] for k in order]
        assert torch.allclose(scores[b].cpu(), torch.tensor([ranked[k][0] for k in order]), rtol=1e-6, atol=0)
    for s in range(1, len(seen.calls)):
        logits, finished = seen.calls[s][0], seen.calls[s][3]
        for b in range(B):
            for k in range(K):
                if finished is not None and bool(finished[b, k]):
                    continue
                tokens = hyps[s - 1][b][k]
                ref = rescored(b, tokens)
                err, size = float((logits[b, k].float() - ref.float()).abs().max()), float(ref.float().abs().max())
                assert err <= 1e-2 * size, (s, b, k, err, size)


def _whisper():
    cfg, sd, x, ids, logits, enc = load_fixture()
    m = W.WhisperForConditionalGenerationQ(transformers.WhisperConfig(**cfg))
    m.load_state_dict(sd)
    return cfg, W.WhisperEngine.from_model(m.half().to(DEV).eval()), x


@pytest.mark.parametrize("beams,prompted,ragged,eos", [(4, False, False, None), (3, True, False, 7), (5, True, True, None), (1, False, False, None)])
def test_whisper(monkeypatch, beams, prompted, ragged, eos):
    cfg, eng, x = _whisper()
    enc = eng.encode(x)
    B, S, _ = enc.shape
    steps = 8
    start = torch.full((B, 1), cfg["decoder_start_token_id"])
    prompt = torch.cat([start, torch.randint(3, 250, (B, 5), generator=torch.Generator().manual_seed(3))], 1) if prompted else start
    lengths = torch.tensor([S - 13 * b for b in range(B)], device=DEV) if ragged else None
    if ragged:
        enc = enc.clone()
        for b in range(B):
            enc[b, int(lengths[b]):] = 30.0  # behind an utterance's states: another's leftovers
    with monkeypatch.context() as patch:
        seen = _Seen(patch)
        if eos is not None:  # a token that does come up ends a hypothesis
            probe = eng.beam_search(enc, steps, beams, prompt if prompted else None, lengths, eos=eos, use_graph=False)[0]
            eos = int(probe[0, 0, 2])
            seen.calls.clear()
        ids, scores = eng.beam_search(enc, steps, beams, prompt if prompted else None, lengths, eos=eos, length_penalty=0.7, use_graph=False)
    eos = cfg["eos_token_id"] if eos is None else eos

    def rescored(b, tokens):
        forced = torch.cat([prompt[b, 1:], torch.tensor(tokens)]).view(-1, 1)
        states = enc[b:b + 1, :int(lengths[b])].contiguous() if ragged else enc[b:b + 1]
        return eng.decode(states, len(forced) + 1, forced_ids=torch.cat([forced, forced[-1:]]), keep_logits=True, use_graph=False)[1][-1, 0]

    _check_search(seen, ids, scores, eos, 0.7, rescored)
    again = eng.beam_search(enc, steps, beams, prompt if prompted else None, lengths, eos=eos, length_penalty=0.7)
    more = eng.beam_search(enc, steps, beams, prompt if prompted else None, lengths, eos=eos, length_penalty=0.7)  # the graph's second use
    for got in (again, more):
        assert torch.equal(got[0], ids) and torch.equal(got[1], scores)
    asrq_b200.check_status()


def test_whisper_refusals():
    cfg, eng, x = _whisper()
    enc = eng.encode(x)
    for kw in (dict(steps=0), dict(steps=33), dict(steps=4, beams=0), dict(steps=4, beams=33), dict(steps=4, prompt=torch.ones(1, 2, dtype=torch.long)),
               dict(steps=30, prompt=torch.ones(enc.shape[0], 4, dtype=torch.long))):
        with pytest.raises(ValueError):
            eng.beam_search(enc, **kw)


@pytest.mark.parametrize("beams,ends", [(4, False), (5, True)])
def test_qwen3(monkeypatch, beams, ends):
    cfg, fm, q = toy_models()
    eng = Q.Qwen3Engine.from_model(q.half().to(DEV))
    B, T, steps, eos = 3, 9, 7, None
    ids0 = torch.randint(0, cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(1))
    emb = fm.model.embed_tokens(ids0).detach().half().to(DEV)
    with monkeypatch.context() as patch:
        seen = _Seen(patch)
        if ends:
            eos = int(eng.beam_search(emb, steps, beams, use_graph=False)[0][1, 0, 3])
            seen.calls.clear()
        ids, scores = eng.beam_search(emb, steps, beams, eos=eos, length_penalty=1.0, use_graph=False)
    eos = BM.end_token(cfg, eos)

    def rescored(b, tokens):
        row = torch.cat([emb[b], eng.embed[torch.tensor(tokens, device=DEV)]]).unsqueeze(0)
        other.prefill(row, 1)
        return other.last_logits[0]

    other = Q.Qwen3Engine.from_model(q)
    _check_search(seen, ids, scores, eos, 1.0, rescored)
    again = eng.beam_search(emb, steps, beams, eos=eos)
    greedy = eng.generate(emb, steps)  # shares the engine's caches
    more = eng.beam_search(emb, steps, beams, eos=eos)
    for got in (again, more):
        assert torch.equal(got[0], ids) and torch.equal(got[1], scores)
    assert greedy.shape == (B, steps)
    asrq_b200.check_status()
