"""The operators of decoding with several hypotheses per utterance, one pass each, on synthetic data of the models' sizes.

    beam_select       the best continuations over the beams and the vocabulary of an utterance
    beam_reorder      the beams' caches follow the hypotheses that were kept
    cross_attention   the rows of an utterance (beams, or the tokens of a prompt) over its encoder states, each of its own length
    prefix_attention  beams or samples of one utterance: the prompt's keys once for all of them, then each one's own

``own`` false: each in elementary torch operations, in 32 bits (the selection, whose order decides, in 64).  ``own`` true: the
library's calls.  ``exact``: the definitions in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# The sizes are those of the models this package runs: Whisper-large-v3 (32 decoder layers, 20 heads of 64, 1500 encoder
# states, 51866 tokens, 448 target positions) and the speech model's Qwen3-1.7B decoder (28 layers, 16 query and 8 key heads of
# 128, 151936 tokens; 20 seconds of audio are 250 states, its prompt 8 tokens).


def listed():
    return [
        # one utterance, five beams: a step's selection, where the latency of a call counts
        dict(name="select 1x5 of 51866", op="select", dtype="fp16", B=1, K=5, V=51866, n=5, finished=0, hidden=0.0),
        # a batch of the speech model; some hypotheses have ended
        dict(name="select 16x5 of 151936", op="select", dtype="bf16", B=16, K=5, V=151936, n=5, finished=2, hidden=0.0),
        # a large batch with twice as many candidates as beams (for a caller that keeps ended ones apart) and suppressed tokens
        dict(name="select 64x8 of 51866", op="select", dtype="fp16", B=64, K=8, V=51866, n=16, finished=0, hidden=0.03),
        # one utterance after 60 tokens: the self-attention caches of all layers
        dict(name="reorder 1x5, 60 of 449", op="reorder", dtype="fp16", L=64, B=1, K=5, H=20, M=449, hd=64, length=60, moved=4, sources=2),
        # a batch after 224 tokens
        dict(name="reorder 8x5, 224 of 449", op="reorder", dtype="fp16", L=64, B=8, K=5, H=20, M=449, hd=64, length=224, moved=3, sources=2),
        # the speech model's own positions behind a shared prompt
        dict(name="reorder 16x5, 100 of 129", op="reorder", dtype="bf16", L=56, B=16, K=5, H=8, M=129, hd=128, length=100, moved=3, sources=2),
        # a step of one utterance with five beams: the window's states are read once for all beams
        dict(name="cross 1x5 on 1500", op="cross", dtype="fp16", B=1, R=5, S=1500, Hq=20, Hkv=20, hd=64, least=1.0),
        # a step of a batch of utterances that are not equally long
        dict(name="cross 16x5 on 150..1500", op="cross", dtype="bf16", B=16, R=5, S=1500, Hq=20, Hkv=20, hd=64, least=0.1),
        # the text before the window as a prompt: many rows at once
        dict(name="cross 16x224 on 1500", op="cross", dtype="fp16", B=16, R=224, S=1500, Hq=20, Hkv=20, hd=64, least=1.0),
        # a step of one utterance with five beams behind 258 prompt positions
        dict(name="prefix 1x5, 258 + 40", op="prefix", dtype="fp16", B=1, K=5, Hq=16, Hkv=8, hd=128, P=258, M=129, shared=40, least=1.0),
        # the same for a batch of 64, as the speech model is served
        dict(name="prefix 64x5, 258 + 65", op="prefix", dtype="bf16", B=64, K=5, Hq=16, Hkv=8, hd=128, P=258, M=129, shared=65, least=1.0),
        # an hour's recording (45000 states), 64 samples of one prompt, each of its own length
        dict(name="prefix 1x64, 45000 + 1..200", op="prefix", dtype="bf16", B=1, K=64, Hq=16, Hkv=8, hd=128, P=45000, M=257, shared=0, least=1.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    dtype, op = rng.choice(["fp16", "bf16"]), rng.choice(["select", "reorder", "cross", "prefix"])
    if op == "select":
        K, V = rng.randint(1, 16), _log(rng, 500, 152000)
        B = _log(rng, 1, max(1, min(64, 80 * 151936 // (K * V))))
        return dict(op=op, dtype=dtype, B=B, K=K, V=V, n=rng.choice([K, min(2 * K, 32)]), finished=rng.randint(0, K // 2), hidden=rng.choice([0.0, 0.1]))
    if op == "reorder":
        K, hd = rng.randint(2, 8), rng.choice([64, 128])
        M, H, L = rng.randint(65, 449), rng.randint(2, 20), 2 * rng.randint(2, 32)
        B = _log(rng, 1, max(1, min(16, 64 * 40 * 20 * 449 * 64 // (L * K * H * M * hd))))
        moved = rng.randint(2, K)
        # moved rows times positions stay below the largest listed case's
        most = max(1, min(M, 64 * 8 * 20 * 224 * 64 * 5 // (L * B * H * hd * 2 * moved)))
        return dict(op=op, dtype=dtype, L=L, B=B, K=K, H=H, M=M, hd=hd, length=_log(rng, 1, most), moved=moved, sources=rng.randint(2, moved))
    hd, Hkv = rng.choice([64, 128]), rng.choice([2, 4, 8, 20])
    group = rng.choice([1, 2]) if Hkv == 20 else rng.choice([1, 2, 4])
    if op == "cross":
        R, S = _log(rng, 1, 448), _log(rng, 17, 6000)
        row = Hkv * group * hd
        B = _log(rng, 1, max(1, min(32, 16 * 224 * 1500 * 1280 // (R * S * row), 16 * 1724 * 1280 // (S * Hkv * hd + R * row))))
        return dict(op=op, dtype=dtype, B=B, R=R, S=S, Hq=Hkv * group, Hkv=Hkv, hd=hd, least=rng.choice([0.0, 0.2, 1.0]))
    K, P, M = rng.randint(1, 16), _log(rng, 1, 45000 * 1024 // (Hkv * hd)), _log(rng, 1, 300)
    B = _log(rng, 1, max(1, min(64, 45000 * 1024 // (P * Hkv * hd + K * M * Hkv * hd))))
    return dict(op=op, dtype=dtype, B=B, K=K, Hq=Hkv * group, Hkv=Hkv, hd=hd, P=P, M=M, shared=rng.choice([0, rng.randint(1, M)]), least=rng.choice([0.0, 0.3, 1.0]))


def _lengths(least, most, count):
    """``count`` lengths from ``least`` of ``most`` to ``most``, evenly spread (the seed shuffles them)."""
    if least >= 1.0:
        return [most] * count
    return [most if count == 1 else round(most * (least + (1 - least) * i / (count - 1))) for i in range(count)]


def _own_lengths(c):
    """The beams' own positions: one for all, or from 1 to four fifths of the room."""
    return [c["shared"]] if c["shared"] else _lengths(min(1.0, 1.25 / c["M"]), max(1, c["M"] * 4 // 5), c["B"] * c["K"])


def prepare(case, seed):
    c, rng = case, random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[c["dtype"]]

    def rnd(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV, dtype=dt) * std

    def ints(values):
        return torch.tensor(values, dtype=torch.int64, device=DEV)

    if c["op"] == "select":
        B, K, V = c["B"], c["K"], c["V"]
        logits = torch.randn(B, K, V, generator=g, device=DEV, dtype=torch.float32) * 2.5
        at = torch.randint(0, V, (B, K, min(V, 12)), generator=g, device=DEV)  # what the model thinks likely
        logits.scatter_reduce_(2, at, torch.rand(at.shape, generator=g, device=DEV) * 12 + 4, "amax")
        if c["hidden"]:  # suppressed tokens
            logits.masked_fill_(torch.rand(V, generator=g, device=DEV) < c["hidden"], float("-inf"))
        scores = -torch.rand(B, K, generator=g, device=DEV).cumsum(1) * 6 - 1
        finished = torch.zeros(B, K, dtype=torch.bool, device=DEV)
        for b in range(B):
            finished[b, rng.sample(range(K), c["finished"])] = True
        return dict(case=c, logits=logits.to(dt), scores=scores, finished=finished if c["finished"] else None, eos=V // 2)
    if c["op"] == "reorder":
        B, K = c["B"], c["K"]
        cache = torch.randn(c["L"], B * K, c["H"], c["M"], c["hd"], generator=g, device=DEV, dtype=dt)
        parents = []
        for _ in range(B):  # `moved` beams take the place of another, from `sources` different ones
            row, beams = list(range(K)), rng.sample(range(K), c["moved"])
            for i, k in enumerate(beams):
                row[k] = beams[(i % c["sources"] + 1) % len(beams)]
            parents.append(row)
        return dict(case=c, cache=cache, parents=ints(parents), length=ints([c["length"]]))
    if c["op"] == "cross":
        B, S, d = c["B"], c["S"], c["Hkv"] * c["hd"]
        kv = rnd(B, S, 2, c["Hkv"], c["hd"])  # a fused projection's output: keys and values side by side
        lengths = _lengths(c["least"], S, B)
        rng.shuffle(lengths)
        return dict(case=c, q=rnd(B, c["R"], c["Hq"], c["hd"], std=1.5), k=kv[:, :, 0], v=kv[:, :, 1], lengths=None if c["least"] >= 1.0 else ints(lengths))
    B, K = c["B"], c["K"]
    prefix = rnd(2, B, c["Hkv"], c["P"], c["hd"])
    suffix = rnd(2, B * K, c["Hkv"], c["M"], c["hd"])
    lengths, mine = _lengths(c["least"], c["P"], B), _own_lengths(c)
    rng.shuffle(lengths)
    rng.shuffle(mine)
    return dict(case=c, q=rnd(B, K, c["Hq"], c["hd"], std=1.5), k_prefix=prefix[0], v_prefix=prefix[1], k_suffix=suffix[0], v_suffix=suffix[1],
                suffix_lengths=ints(mine), prefix_lengths=None if c["least"] >= 1.0 else ints(lengths))


def _select(logits, scores, n, finished, eos):
    B, K, V = logits.shape
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    norm = top + (x - top).exp().sum(-1, keepdim=True).log()
    some = torch.isfinite(top)
    at = torch.arange(V, device=x.device)
    if finished is not None:  # an ended hypothesis goes on as it is
        over = finished.unsqueeze(-1)
        x = torch.where(over, torch.where(at == eos, 0.0, float("-inf")), x)
        norm, some = torch.where(over, 0.0, norm), some | over
    some = some & torch.isfinite(scores).unsqueeze(-1)
    x, norm = torch.where(some, x, float("-inf")), torch.where(some, norm, 0.0)
    # within a beam by logit, then by index: one whole number for both
    bits = (x.float() + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7fffffff, bits)
    key = (bits * (1 << 32) + (V - 1 - at)).topk(min(n, V), dim=-1).values
    token = V - 1 - (key & 0xffffffff)
    cand = scores.double().unsqueeze(-1) + (x.gather(-1, token) - norm)
    cand = torch.where(some, cand, float("-inf"))
    flat = (torch.arange(K, device=x.device).view(1, K, 1) * V + token).reshape(B, -1)
    by_place = flat.argsort(-1)
    flat, cand = flat.gather(-1, by_place), cand.reshape(B, -1).gather(-1, by_place)
    best = torch.sort(cand, dim=-1, descending=True, stable=True).indices[:, :n]
    flat, cand = flat.gather(-1, best), cand.gather(-1, best)
    parents, tokens = flat // V, flat % V
    out = (cand.float(), parents, tokens)
    return out if finished is None else out + (finished.gather(1, parents) | (tokens == eos),)


def _reorder(cache, parents, length):
    B, K = parents.shape
    rows = (torch.arange(B, device=parents.device).unsqueeze(1) * K + parents).reshape(-1)
    cache[:, :, :, :length] = cache[:, :, :, :length].index_select(1, rows)
    return cache


def _softmax(s, mask):
    s = s.masked_fill(~mask, float("-inf"))
    top = s.amax(-1, keepdim=True)
    e = (s - torch.where(torch.isfinite(top), top, 0.0)).exp()
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _cross(q, k, v, lengths):
    B, R, Hq, hd = q.shape
    S, Hkv = k.shape[1:3]
    rows = q.float().view(B, R, Hkv, Hq // Hkv, hd).permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, hd)
    s = rows @ k.float().permute(0, 2, 3, 1) * hd ** -0.5
    mask = torch.ones(B, 1, 1, S, dtype=torch.bool, device=q.device) if lengths is None else \
        torch.arange(S, device=q.device).view(1, 1, 1, S) < lengths.view(B, 1, 1, 1)
    o = _softmax(s, mask) @ v.float().permute(0, 2, 1, 3)
    return o.view(B, Hkv, R, Hq // Hkv, hd).permute(0, 2, 1, 3, 4).reshape(B, R, Hq, hd).to(q.dtype)


def _prefix(q, k_prefix, v_prefix, k_suffix, v_suffix, suffix_lengths, prefix_lengths):
    B, K, Hq, hd = q.shape
    Hkv, P = k_prefix.shape[1:3]
    M, G = k_suffix.shape[2], Hq // Hkv
    rows = q.float().view(B, K, Hkv, G, hd).permute(0, 2, 1, 3, 4)  # B, Hkv, K, G, hd
    first = (rows.reshape(B, Hkv, K * G, hd) @ k_prefix.float().transpose(-1, -2)).view(B, Hkv, K, G, P)
    mine = rows @ k_suffix.float().view(B, K, Hkv, M, hd).permute(0, 2, 1, 4, 3)
    at = torch.arange(P, device=q.device).expand(B, P) < (P if prefix_lengths is None else prefix_lengths.view(B, 1))
    own_at = torch.arange(M, device=q.device) < suffix_lengths.view(-1, 1)
    mask = torch.cat([at.view(B, 1, 1, 1, P).expand(B, 1, K, 1, P), own_at.expand(B * K, M).reshape(B, 1, K, 1, M)], -1)
    p = _softmax(torch.cat([first, mine], -1) * hd ** -0.5, mask)
    o = (p[..., :P].reshape(B, Hkv, K * G, P) @ v_prefix.float()).view(B, Hkv, K, G, hd)
    o = o + p[..., P:] @ v_suffix.float().view(B, K, Hkv, M, hd).permute(0, 2, 1, 3, 4)
    return o.permute(0, 2, 1, 3, 4).reshape(B, K, Hq, hd).to(q.dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        import asrq_b200
        if c["op"] == "select":
            return asrq_b200.beam_select(s["logits"], s["scores"], c["n"], finished=s["finished"], eos=s["eos"] if s["finished"] is not None else None)
        if c["op"] == "reorder":
            return asrq_b200.beam_reorder(s["cache"], s["parents"], s["length"])
        if c["op"] == "cross":
            return asrq_b200.cross_attention(s["q"], s["k"], s["v"], lengths=s["lengths"])
        return asrq_b200.prefix_attention(s["q"], s["k_prefix"], s["v_prefix"], s["k_suffix"], s["v_suffix"], s["suffix_lengths"],
                                          prefix_lengths=s["prefix_lengths"])
    if c["op"] == "select":
        return _select(s["logits"], s["scores"], c["n"], s["finished"], s["eos"])
    if c["op"] == "reorder":
        return _reorder(s["cache"], s["parents"], c["length"])
    if c["op"] == "cross":
        return _cross(s["q"], s["k"], s["v"], s["lengths"])
    return _prefix(s["q"], s["k_prefix"], s["v_prefix"], s["k_suffix"], s["v_suffix"], s["suffix_lengths"], s["prefix_lengths"])


def work(case):
    c = case
    if c["op"] == "select":  # the logits of the hypotheses that go on; four operations a value for the normalisation
        values = c["B"] * (c["K"] - c["finished"]) * c["V"]
        return {"bytes": 2 * values + c["B"] * (4 * c["K"] + 20 * c["n"]), "flops": 4 * values}
    if c["op"] == "reorder":  # rows that move are written, those they come from read
        return {"bytes": 2 * c["L"] * c["B"] * c["H"] * c["length"] * c["hd"] * (c["moved"] + c["sources"]) + 8 * c["B"] * c["K"], "flops": 0}
    if c["op"] == "cross":
        keys = sum(_lengths(c["least"], c["S"], c["B"]))
        return {"bytes": 4 * (c["B"] * c["R"] * c["Hq"] + keys * c["Hkv"]) * c["hd"], "flops": 4 * c["R"] * c["Hq"] * c["hd"] * keys}
    shared, mine = sum(_lengths(c["least"], c["P"], c["B"])), _own_lengths(c)
    mine = sum(mine) * (c["B"] * c["K"] if len(mine) == 1 else 1)
    return {"bytes": 4 * (c["B"] * c["K"] * c["Hq"] + (shared + mine) * c["Hkv"]) * c["hd"], "flops": 4 * (shared * c["K"] + mine) * c["Hq"] * c["hd"]}


def _attend64(q, keys, values, scale):
    """One sequence: q (rows, Hkv, G, hd), keys and values (n, Hkv, hd), all in 64 bits."""
    if keys.shape[0] == 0:
        return torch.zeros_like(q)
    w = torch.softmax(torch.einsum("rhgd,nhd->rhgn", q, keys) * scale, -1)
    return torch.einsum("rhgn,nhd->rhgd", w, values)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "reorder":
        return None  # copies: nothing is computed
    if c["op"] == "select":
        K, V = c["K"], c["V"]
        best, parents, tokens = [], [], []
        for b in range(c["B"]):
            table = torch.full((K, V), float("-inf"), dtype=torch.float64, device=DEV)
            for k in range(K):
                score = s["scores"][b, k].double()
                if s["finished"] is not None and bool(s["finished"][b, k]):
                    table[k, s["eos"]] = score
                else:
                    x = s["logits"][b, k].double()
                    table[k] = score + x - torch.logsumexp(x, 0)
            order = torch.sort(table.view(-1), descending=True, stable=True)
            best.append(order.values[:c["n"]])
            parents.append(order.indices[:c["n"]] // V)
            tokens.append(order.indices[:c["n"]] % V)
        out = (torch.stack(best), torch.stack(parents), torch.stack(tokens))
        return out if s["finished"] is None else out + (None,)
    hd, scale = c["hd"], 1.0 / math.sqrt(c["hd"])
    out = []
    if c["op"] == "cross":
        for b in range(c["B"]):
            n = c["S"] if s["lengths"] is None else int(s["lengths"][b])
            q = s["q"][b].double().view(c["R"], c["Hkv"], -1, hd)
            out.append(_attend64(q, s["k"][b, :n].double(), s["v"][b, :n].double(), scale))
        return torch.stack(out).view(c["B"], c["R"], c["Hq"], hd)
    mine = s["suffix_lengths"].tolist()
    for b in range(c["B"]):
        n = c["P"] if s["prefix_lengths"] is None else int(s["prefix_lengths"][b])
        kp, vp = (s[name][b, :, :n].double().transpose(0, 1) for name in ("k_prefix", "v_prefix"))
        for i in range(b * c["K"], (b + 1) * c["K"]):
            m = mine[i % len(mine)]
            ks, vs = (s[name][i, :, :m].double().transpose(0, 1) for name in ("k_suffix", "v_suffix"))
            q = s["q"][b, i - b * c["K"]].double().view(1, c["Hkv"], -1, hd)
            out.append(_attend64(q, torch.cat([kp, ks]), torch.cat([vp, vs]), scale)[0])
    return torch.stack(out).view(c["B"], c["K"], c["Hq"], hd)
