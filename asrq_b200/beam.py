"""Decoding with several hypotheses (beams) per utterance: the operators of a step (csrc/beam.cu, csrc/rows_attn.cu).

The reference decodes with the stock models' ``generate`` (asrq/evaluation/openasr.py), where beam search ranks the continuations and reorders
the caches by a chain of tensor operations, and holds the prompt's keys and the encoder's once per beam.  Here

* :func:`beam_select` ranks the continuations of a step, :func:`beam_reorder` lets the caches follow them;
* :func:`cross_attention` reads an utterance's encoder states once for all its beams, or for the tokens of a prompt;
* :func:`prefix_attention` reads a prompt's keys once for all beams or samples behind it.

``WhisperEngine.beam_search`` and ``Qwen3Engine.beam_search`` run them.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from . import linear as _linear
from .linear import _call_scratch, _expect, _on_device, _require_cuda_16bit, _workspace


def _ints(t: torch.Tensor, like: torch.Tensor) -> bool:
    return t.dtype == torch.int64 and t.device == like.device


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: int = None, finished: torch.Tensor = None, eos: int = None):
    """The ``n`` (by default as many as beams) best continuations of every utterance over its beams and the vocabulary:
    ``scores[b, k] + log_softmax(logits[b, k])[v]``, descending, of equal ones the lowest ``k * V + v``.

    ``logits`` (B, K, V) 16-bit with contiguous rows, ``scores`` (B, K) fp32.  Returns ``(scores, parents, tokens)`` of shape (B, n): fp32 and
    int64, ``parents`` the beam that goes on.  A beam's normalisation has exponentials of 32 bits (within 4e-6): candidates of different beams that lie nearer than
    8e-6 may come in either order.  With ``finished`` (B, K) bool and ``eos``: a finished beam goes on with ``eos`` at its own score
    and nothing else, and the fourth result says which of the new hypotheses have ended.  A beam whose score is not finite (at the first
    step all but one) or whose logits are no distribution (a NaN, a +inf, nothing above -inf) offers its tokens at -inf."""
    if _linear._native is not None:  # the ordinary case in native code; None where it is not one
        out = _linear._native.beam_select(logits, scores, scores.shape[-1] if n is None else n, finished, eos)
        if out is not None:
            return out
    dt = _require_cuda_16bit(logits, "beam_select")
    _expect(logits.dim() == 3, f"beam_select: logits (B, K, V), got {tuple(logits.shape)}")
    B, K, V = logits.shape
    n = K if n is None else int(n)
    _expect(scores.dtype == torch.float32 and scores.device == logits.device and tuple(scores.shape) == (B, K) and (finished is None) == (eos is None) and
            (finished is None or (finished.dtype == torch.bool and finished.device == logits.device and tuple(finished.shape) == (B, K))),
            "beam_select: scores fp32 (B, K), finished bool (B, K) with eos, on the logits' device")
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    finished = None if finished is None else finished.contiguous()
    dev = logits.device
    out = torch.empty((B, n), dtype=torch.float32, device=dev)
    picked = torch.empty((2, B, n), dtype=torch.int64, device=dev)
    over = None if finished is None else torch.empty((B, n), dtype=torch.bool, device=dev)
    if B:
        with _on_device(dev):
            _lib.call("asrq_beam_select", logits.data_ptr(), logits.stride(0), logits.stride(1), scores.data_ptr(), None if over is None else finished.data_ptr(),
                      0 if eos is None else int(eos), out.data_ptr(), picked[0].data_ptr(), picked[1].data_ptr(), None if over is None else over.data_ptr(),
                      B, K, V, n, dt, torch.cuda.current_stream(dev).cuda_stream)
    return (out, picked[0], picked[1]) if over is None else (out, picked[0], picked[1], over)


def beam_reorder(cache: torch.Tensor, parents: torch.Tensor, length) -> torch.Tensor:
    """The beams' caches follow the hypotheses that were kept, in place: ``cache`` (L, B * K, heads, max_len, head_dim), contiguous, of any type with
    16-byte positions; for every utterance b and beam k the positions below ``length`` (an int, or a one-element int64 CUDA tensor)
    become those of beam ``parents[b, k]`` (``parents`` (B, K) int64); a parent that is no beam leaves the row as it is.  Returns ``cache``."""
    if _linear._native is not None and _linear._native.beam_reorder(cache, parents, length):
        return cache
    if not cache.is_cuda:
        raise RuntimeError(f"beam_reorder: cache is on {cache.device}; asrq_b200 runs on CUDA (sm_100a) only and has no CPU path")
    _expect(cache.dim() == 5 and cache.is_contiguous() and parents.dim() == 2 and parents.numel() == cache.shape[1] and _ints(parents, cache),
            f"beam_reorder: contiguous cache (L, B * K, heads, max_len, head_dim) and int64 parents (B, K) (cache {tuple(cache.shape)}, parents "
            f"{tuple(parents.shape)})")
    on_dev = isinstance(length, torch.Tensor)
    _expect(not on_dev or (length.numel() == 1 and _ints(length, cache)), "beam_reorder: length is an int or one int64 on the cache's device")
    L, _, H, M, hd = cache.shape
    if cache.numel() == 0:
        return cache
    parents = parents.contiguous()
    with _on_device(cache.device):
        ws = _workspace(cache.device, _lib.STATUS_BYTES)
        _lib.call("asrq_beam_reorder", cache.data_ptr(), parents.data_ptr(), length.data_ptr() if on_dev else None, 0 if on_dev else int(length), L,
                  parents.shape[0], parents.shape[1], H, M, hd * cache.element_size(), ws.data_ptr(), ws.numel(),
                  torch.cuda.current_stream(cache.device).cuda_stream)
    return cache


def _strided(x: torch.Tensor) -> torch.Tensor:
    """As it is where the kernels can read it (aligned vectors of 8 along the last dimension), else a copy."""
    if x.stride(3) == 1 and x.data_ptr() % 16 == 0 and all(x.stride(i) % 8 == 0 or x.shape[i] == 1 for i in range(3)):
        return x
    return x.clone(memory_format=torch.contiguous_format)


def _strides(x: torch.Tensor, *dims: int):
    return (ctypes.c_int64 * 3)(*(x.stride(d) if x.shape[d] > 1 else 0 for d in dims))


def _memory(q: torch.Tensor, key_heads: int, shared: int, own: int):
    """(workspace, its bytes, scratch, its bytes) of a call."""
    ws = _workspace(q.device, _lib.STATUS_BYTES)
    need = int(_lib.load().asrq_rows_attention_scratch_bytes(q.shape[0], q.shape[1], q.shape[2], key_heads, q.shape[3], shared, own))
    scratch = _call_scratch(need, q.device)
    return ws, ws.data_ptr(), ws.numel(), scratch, None if scratch is None else scratch.data_ptr(), 0 if scratch is None else need


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor = None, scale: float = None) -> torch.Tensor:
    """Attention of the rows of an utterance (the beams of a step, or the tokens of a prompt) over its encoder states: ``q`` (B, R, heads,
    head_dim), ``k`` and ``v`` (B, S, key heads, head_dim), 16-bit, any strides with contiguous heads (``kv.view(B, S, 2, heads, head_dim)[:, :, i]`` of a
    fused projection); ``lengths`` (B,) int64 on the device, None for S everywhere.  ``scale`` head_dim ** -0.5 by default.  Returns (B, R, heads,
    head_dim); a row without keys is zero."""
    if _linear._native is not None:
        out = _linear._native.cross_attention(q, k, v, lengths, scale)
        if out is not None:
            return out
    dt = _require_cuda_16bit(q, "cross_attention")
    _expect(q.dim() == k.dim() == 4 and v.shape == k.shape, f"cross_attention: q (B, R, heads, head_dim), k and v (B, S, key heads, head_dim), got "
            f"{tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, R, Hq, hd = q.shape
    S, Hkv = k.shape[1], k.shape[2]
    _expect(k.shape[0] == B and k.shape[3] == hd and Hkv > 0 and Hq % Hkv == 0 and all(t.dtype == q.dtype and t.device == q.device for t in (k, v)) and
            (lengths is None or (tuple(lengths.shape) == (B,) and _ints(lengths, q))),
            f"cross_attention: tensors of one type on one device, heads a multiple of the key heads, int64 lengths (B,) (q {tuple(q.shape)}, k {tuple(k.shape)})")
    q, k, v = _strided(q), _strided(k), _strided(v)
    lengths = None if lengths is None else lengths.contiguous()
    out = torch.empty((B, R, Hq, hd), dtype=q.dtype, device=q.device)
    if out.numel():
        with _on_device(q.device):
            ws, ws_ptr, ws_bytes, scratch, scratch_ptr, need = _memory(q, Hkv, S, 0)
            _lib.call("asrq_cross_attention", q.data_ptr(), _strides(q, 0, 1, 2), k.data_ptr(), _strides(k, 0, 2, 1), v.data_ptr(), _strides(v, 0, 2, 1),
                      None if lengths is None else lengths.data_ptr(), out.data_ptr(), B, R, Hq, Hkv, hd, S, hd ** -0.5 if scale is None else float(scale),
                      dt, ws_ptr, ws_bytes, scratch_ptr, need, torch.cuda.current_stream(q.device).cuda_stream)
    return out


def prefix_attention(q: torch.Tensor, k_prefix: torch.Tensor, v_prefix: torch.Tensor, k_suffix: torch.Tensor, v_suffix: torch.Tensor,
                     suffix_lengths: torch.Tensor, prefix_lengths: torch.Tensor = None, scale: float = None) -> torch.Tensor:
    """Attention of one decoding step of K beams (or samples) per utterance behind a prompt that they share: ``q`` (B, K, heads, head_dim); the
    prompt's keys and values once per utterance, (B, key heads, P, head_dim); each beam's own, (B * K, key heads, M, head_dim).  ``suffix_lengths``
    int64 on the device: one for all beams, or B * K; ``prefix_lengths`` (B,) int64, None for P everywhere.  Returns (B, K, heads, head_dim); a
    row without keys is zero."""
    if _linear._native is not None:
        out = _linear._native.prefix_attention(q, k_prefix, v_prefix, k_suffix, v_suffix, suffix_lengths, prefix_lengths, scale)
        if out is not None:
            return out
    dt = _require_cuda_16bit(q, "prefix_attention")
    _expect(q.dim() == k_prefix.dim() == k_suffix.dim() == 4 and v_prefix.shape == k_prefix.shape and v_suffix.shape == k_suffix.shape,
            "prefix_attention: q (B, K, heads, head_dim), prefix (B, key heads, P, head_dim), suffix (B * K, key heads, M, head_dim)")
    B, K, Hq, hd = q.shape
    Hkv, P, M = k_prefix.shape[1], k_prefix.shape[2], k_suffix.shape[2]
    _expect(k_prefix.shape[0] == B and k_prefix.shape[3] == hd and Hkv > 0 and Hq % Hkv == 0 and tuple(k_suffix.shape) == (B * K, Hkv, M, hd) and
            all(t.dtype == q.dtype and t.device == q.device for t in (k_prefix, v_prefix, k_suffix, v_suffix)) and
            suffix_lengths.numel() in (1, B * K) and _ints(suffix_lengths, q) and
            (prefix_lengths is None or (tuple(prefix_lengths.shape) == (B,) and _ints(prefix_lengths, q))),
            f"prefix_attention: tensors of one type on one device; q {tuple(q.shape)}, prefix {tuple(k_prefix.shape)}, suffix {tuple(k_suffix.shape)}, int64 lengths, "
            "one or B * K of the suffix, B of the prefix")
    q, k_prefix, v_prefix, k_suffix, v_suffix = (_strided(t) for t in (q, k_prefix, v_prefix, k_suffix, v_suffix))
    suffix_lengths = suffix_lengths.contiguous()
    prefix_lengths = None if prefix_lengths is None else prefix_lengths.contiguous()
    out = torch.empty((B, K, Hq, hd), dtype=q.dtype, device=q.device)
    if out.numel():
        with _on_device(q.device):
            ws, ws_ptr, ws_bytes, scratch, scratch_ptr, need = _memory(q, Hkv, P, M)
            _lib.call("asrq_prefix_attention", q.data_ptr(), _strides(q, 0, 1, 2), k_prefix.data_ptr(), _strides(k_prefix, 0, 1, 2), v_prefix.data_ptr(),
                      _strides(v_prefix, 0, 1, 2), None if prefix_lengths is None else prefix_lengths.data_ptr(), k_suffix.data_ptr(), _strides(k_suffix, 0, 1, 2),
                      v_suffix.data_ptr(), _strides(v_suffix, 0, 1, 2), suffix_lengths.data_ptr(), suffix_lengths.numel(), out.data_ptr(), B, K, Hq, Hkv, hd, P, M,
                      hd ** -0.5 if scale is None else float(scale), dt, ws_ptr, ws_bytes, scratch_ptr, need,
                      torch.cuda.current_stream(q.device).cuda_stream)
    return out


def end_token(config, eos=None):
    """The token that ends a hypothesis: the one given, else the configuration's (the first of several), None where it has none."""
    eos = getattr(config, "eos_token_id", None) if eos is None else eos
    eos = next(iter(eos), None) if isinstance(eos, (list, tuple)) else eos
    return None if eos is None else int(eos)


class BeamState:
    """The hypotheses of a batch while they grow: B utterances, K beams each, ``steps`` tokens.  :meth:`start` takes the logits of the prompt's last position
    (one hypothesis per utterance), :meth:`advance` those of a step; both leave the next tokens in ``tok`` (B * K,).  Everything lives in static
    buffers and every index on the device, so :meth:`advance` may be captured.  An ended hypothesis is carried along with the end token
    (``eos``; None: nothing ends) at its score; what is kept of a step are tokens and parents, from which :meth:`hypotheses` reads the sequences
    back."""

    def __init__(self, batch: int, beams: int, steps: int, eos, device):
        self.B, self.K, self.steps, self.eos = batch, beams, steps, eos
        self.tok = torch.zeros(batch * beams, dtype=torch.long, device=device)
        self.at = torch.zeros(1, dtype=torch.long, device=device)  # tokens so far
        self.scores = torch.zeros(batch, beams, dtype=torch.float32, device=device)
        self.finished = torch.zeros(batch, beams, dtype=torch.bool, device=device)
        self.tokens = torch.zeros(steps, batch, beams, dtype=torch.long, device=device)
        self.parents = torch.zeros(steps, batch, beams, dtype=torch.long, device=device)

    def start(self, logits: torch.Tensor) -> None:
        """``logits`` (B, V): the K best tokens of every utterance open its beams (the vocabulary has as many)."""
        scores, parents, tokens = beam_select(logits.view(self.B, 1, -1), torch.zeros(self.B, 1, dtype=torch.float32, device=logits.device), self.K)
        self.tokens[0], self.parents[0] = tokens, parents
        self.scores.copy_(scores)
        if self.eos is not None:
            self.finished.copy_(tokens == self.eos)
        self.tok.copy_(tokens.view(-1))
        self.at.fill_(1)

    def advance(self, logits: torch.Tensor, caches, length: torch.Tensor) -> None:
        """``logits`` (B * K, V): selects, and lets the ``caches`` (each as :func:`beam_reorder` takes it) follow up to ``length`` positions."""
        picked = beam_select(logits.view(self.B, self.K, -1), self.scores, finished=None if self.eos is None else self.finished, eos=self.eos)
        scores, parents, tokens = picked[:3]
        for cache in caches:
            beam_reorder(cache, parents, length)
        self.scores.copy_(scores)
        if self.eos is not None:
            self.finished.copy_(picked[3])
        self.tok.copy_(tokens.view(-1))
        self.tokens.index_copy_(0, self.at, tokens.unsqueeze(0))
        self.parents.index_copy_(0, self.at, parents.unsqueeze(0))
        self.at.add_(1)

    def hypotheses(self, length_penalty: float = 1.0):
        """``(ids, scores)``: ids (B, K, steps), the end token behind the end; scores (B, K): the sum of the log probabilities over the number of
        tokens, the end token among them, to the power of ``length_penalty``.  Best first."""
        ids = torch.empty(self.B, self.K, self.steps, dtype=torch.long, device=self.tok.device)
        beam = torch.arange(self.K, device=self.tok.device).expand(self.B, self.K)
        for s in range(self.steps - 1, -1, -1):
            ids[:, :, s] = self.tokens[s].gather(1, beam)
            beam = self.parents[s].gather(1, beam)
        length = ids.new_full((self.B, self.K), self.steps) if self.eos is None else ((ids == self.eos).cumsum(-1) <= (ids == self.eos)).sum(-1)  # up to the first end token
        scores = self.scores / length.to(torch.float32) ** length_penalty
        order = torch.sort(scores, dim=1, descending=True, stable=True)
        return ids.gather(1, order.indices.unsqueeze(-1).expand_as(ids)), order.values
