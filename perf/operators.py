"""Operators of a serving step over many requests, as cases that can be timed and compared.

Requests share a model's projections but not their fine-tunes, and a step may carry several drafted tokens per request:

* ``adapt``: every stream's low-rank adapter is added beside 1 to 3 shared projections (``ops.adapt_rows``),
  ``y + scale[id] * (x A[id]^T) B[id]^T`` for the rows of a stream with adapter ``id``, ``y`` for streams without one;
* ``verify``: drafted tokens are accepted or replaced by the target's probabilities (``ops.verify_drafts``), so that what
  comes out is distributed as if the target had drawn every token;
* ``advance``: the recurrent state of every stream moves on over as many of the step's tokens as were accepted
  (``ops.advance_state``).

Each has a plain form of elementary torch operations and, where ``own`` is set, the framework's call.
"""
from __future__ import annotations

import math

import torch

from rwkvstic_b200.synth import SHAPES, VOCAB

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ITEM = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5                      # of the layer norms


# ---------------------------------------------------------------------------------------------- the cases
def _adapt(name, embed, site, streams, tokens, rank, adapters, weights, rows):
    return {"name": name, "op": "adapt", "embed": embed, "site": site, "streams": streams, "tokens": tokens, "rank": rank,
            "adapters": adapters, "weights": weights, "rows": rows}


def _verify(name, streams, drafts, vocab, draft_probs, ragged):
    return {"name": name, "op": "verify", "streams": streams, "drafts": drafts, "vocab": vocab, "draft_probs": draft_probs,
            "ragged": ragged}


def _advance(name, shape, streams, tokens):
    layers, embed = SHAPES[shape]
    return {"name": name, "op": "advance", "layers": layers, "embed": embed, "streams": streams, "tokens": tokens}


def listed():
    return [
        # One user's token loop with a fine-tune of their own: key, value and receptance of a block, where latency counts.
        _adapt("adapt_1b5_kvr_1", 2048, "kvr", 1, 1, 16, 8, "bf16", "fp32"),
        # A server's step over many sessions that share 48 fine-tunes: the bytes of the adapters in use.
        _adapt("adapt_7b_ffn_64", 4096, "ffn", 64, 1, 16, 48, "fp16", "fp32"),
        # The same with the whole capacity in use, adapters of their own for most, and activations held in 16 bits.
        _adapt("adapt_7b_kvr_256", 4096, "kvr", 256, 1, 32, 200, "bf16", "bf16"),
        # Five drafted rows for each of 48 sessions through the logits' projection, whose rows have an odd length.
        _adapt("adapt_3b_head_48x5", 2560, "head", 48, 5, 8, 20, "bf16", "fp32"),
        # Unquantised fp32 weights with fp32 adapters, a short prompt.
        _adapt("adapt_169m_out_fp32_37", 768, "out", 1, 37, 12, 4, "fp32", "fp32"),
        # Two prompts of odd length, all in 16 bits; then a batch of long documents, the largest call.
        _adapt("adapt_3b_value_2x701", 2560, "value", 2, 701, 32, 3, "fp16", "fp16"),
        _adapt("adapt_3b_ffn_8x1024", 2560, "ffn", 8, 1024, 64, 6, "bf16", "fp32"),
        # Drafts of one user; of a server's sessions, each with as many as its draft model was sure of; of all its capacity,
        # proposed by looking up earlier text, which gives tokens and no probabilities.
        _verify("verify_1x4", 1, 4, VOCAB, True, False),
        _verify("verify_64x5_ragged", 64, 5, VOCAB, True, True),
        _verify("verify_256x7_lookup", 256, 7, VOCAB, False, True),
        # After one user's draft on the smallest model; after a server's on the headline model.
        _advance("advance_169m_1x5", "169m", 1, 5),
        _advance("advance_7b_64x6", "7b", 64, 6),
    ]


def _spread(rng, lo, hi):
    """A whole number from lo to hi, uniform in its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["adapt"] * 5 + ["verify"] * 3 + ["advance"] * 2)
    if op == "verify":
        drafts, vocab = rng.randint(1, 12), VOCAB if rng.random() < 0.5 else _spread(rng, 200, 70000)
        most = 256 * 8 * VOCAB // ((2 * drafts + 1) * vocab)          # no more work than the largest listed one
        return {"op": op, "streams": _spread(rng, 1, min(256, most)), "drafts": drafts, "vocab": vocab,
                "draft_probs": rng.random() < 0.7, "ragged": rng.random() < 0.5}
    if op == "advance":
        layers, embed = rng.choice(list(SHAPES.values())) if rng.random() < 0.5 else (rng.randint(1, 40), 128 * _spread(rng, 2, 40))
        tokens = _spread(rng, 1, 24)
        most = 32 * 4096 * 64 * 6 // (layers * embed * max(tokens, 4))
        return {"op": op, "layers": layers, "embed": embed, "streams": _spread(rng, 1, max(1, min(256, most))), "tokens": tokens}
    embed = rng.choice([e for _, e in SHAPES.values()]) if rng.random() < 0.5 else 128 * _spread(rng, 2, 40)
    site = rng.choice(["kvr", "out", "ffn", "value", "head"])
    weights = rng.choice(["bf16"] * 3 + ["fp16"] * 2 + ["fp32"])
    rows = weights if rng.random() < 0.4 else "fp32"
    rank = rng.choice([4, 8, 8, 12, 16, 16, 20, 32, 32, 48, 64, 64, 100, 128])
    k, outs = _site(embed, site)
    largest = 8192 * (2560 + 2 * 10240 + 2560 + 2 * 2560), 8192 * 64 * (4 * 2560 + 10240)   # values moved, products: the listed one's
    most = min(8192, largest[0] // (k * len(outs) + 2 * sum(outs)), largest[1] // (rank * (k * len(outs) + sum(outs))))
    if rng.random() < 0.6:                                          # a decoding step, with or without drafts
        tokens = 1 if rng.random() < 0.6 else rng.randint(2, 9)
        streams = _spread(rng, 1, min(256, most // tokens))
    else:                                                           # prompts
        streams = 1 if rng.random() < 0.5 else rng.randint(2, 8)
        tokens = _spread(rng, 2, min(2048, most // streams))
    return {"op": op, "embed": embed, "site": site, "streams": streams, "tokens": tokens, "rank": rank,
            "adapters": _spread(rng, 1, 200 if rank <= 32 else 40), "weights": weights, "rows": rows}


def _site(embed, site):
    """Inputs and outputs of the projections that an adapter call stands beside."""
    ffn = 4 * embed
    return {"kvr": (embed, [embed] * 3), "out": (embed, [embed]), "ffn": (embed, [ffn, embed]), "value": (ffn, [embed]),
            "head": (embed, [VOCAB])}[site]


# ---------------------------------------------------------------------------------------------- inputs
def _ids(case, g):
    """One adapter per stream, as evenly as they go round; every eighth stream has none."""
    streams = case["streams"]
    ids = torch.arange(streams, device=DEVICE) % case["adapters"]
    ids[streams - streams // 8:] = -1
    return ids[torch.randperm(streams, generator=g, device=DEVICE)]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device=DEVICE) * std).to(dtype)

    if case["op"] == "adapt":
        k, outs = _site(case["embed"], case["site"])
        n, r, rows, w, t = case["adapters"], case["rank"], case["streams"] * case["tokens"], DTYPES[case["weights"]], DTYPES[case["rows"]]
        # the adapter's share of an output is some tenths of the projection's own
        banks = [(normal(n, r, k, std=k ** -0.5, dtype=w), normal(n, o, r, std=0.3 * r ** -0.5, dtype=w),
                  0.5 + torch.rand(n, generator=g, device=DEVICE)) for o in outs]
        ys = [normal(rows, o, dtype=t) for o in outs]
        return {"case": case, "banks": banks, "ids": _ids(case, g), "xs": [normal(rows, k, dtype=t) for _ in outs], "ys": ys,
                "outs": [torch.empty_like(y) for y in ys]}
    if case["op"] == "verify":
        B, K, V = case["streams"], case["drafts"], case["vocab"]
        # distributions with one likely token (a few percent to nine tenths) whose unlikely ones a sampler has cut off, so that
        # they do not sum to one; the draft's resemble them
        logits = normal(B, K + 1, V, std=3.0)
        likely = torch.randint(0, V, (B, K + 1, 1), generator=g, device=DEVICE)
        logits.scatter_(2, likely, math.log(V) + 1.5 + 6.0 * torch.rand(B, K + 1, 1, generator=g, device=DEVICE))
        cut = lambda p: torch.where(p > 0.02 / V, p, torch.zeros_like(p))
        target = cut(torch.softmax(logits, -1))
        draft = cut(torch.softmax(logits[:, :K] + normal(B, K, V, std=0.7), -1))
        tokens = torch.multinomial(draft.reshape(B * K, V), 1, generator=g).reshape(B, K)
        lengths = torch.randint(0, K + 1, (B,), generator=g, device=DEVICE) if case["ragged"] else None
        return {"case": case, "target": target, "draft": draft if case["draft_probs"] else None, "tokens": tokens,
                "u": torch.rand(B, K + 1, generator=g, device=DEVICE), "lengths": lengths}
    L, C, B, T = case["layers"], case["embed"], case["streams"], case["tokens"]
    state = normal(B, L, 5, C)
    state[:, :, 3] = 1.0 + 9.0 * torch.rand(B, L, C, generator=g, device=DEVICE)
    state[:, :, 2] *= state[:, :, 3]
    trace = normal(L, 4, B, T, C)
    trace[:, :2] += 0.3
    params = normal(L, 5, C)
    params[:, 0] = 1.0 + 0.1 * params[:, 0]
    params[:, 2] = 1.0 + 0.1 * params[:, 2]
    params[:, 4] = -torch.exp(torch.rand(L, C, generator=g, device=DEVICE) * 8.0 - 5.0)     # decays of the synthetic checkpoints
    counts = torch.randint(1, T + 1, (B,), generator=g, device=DEVICE)
    return {"case": case, "state": state, "counts": counts, "trace": trace, "params": params, "out": torch.empty_like(state)}


# ---------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if case["op"] == "adapt":
        if own:
            from rwkvstic_b200 import ops
            return ops.adapt_rows(state["banks"], state["xs"], state["ids"], state["ys"], state["outs"])
        return [_plain_adapt(a, b, s, x, state["ids"], y) for (a, b, s), x, y in zip(state["banks"], state["xs"], state["ys"])]
    if case["op"] == "verify":
        if own:
            from rwkvstic_b200 import ops
            return ops.verify_drafts(state["target"], state["draft"], state["tokens"], state["u"], state["lengths"])
        return _plain_verify(state["target"], state["draft"], state["tokens"], state["u"], state["lengths"])
    if own:
        from rwkvstic_b200 import ops
        return ops.advance_state(state["state"], state["counts"], state["trace"], state["params"], state["out"])
    return _plain_advance(state["state"], state["counts"], state["trace"], state["params"])


def _plain_adapt(a, b, scale, x, ids, y):
    streams, rows = ids.shape[0], x.shape[0]
    has, at = ids >= 0, ids.clamp(min=0)
    h = torch.bmm(x.float().reshape(streams, rows // streams, -1), a[at].float().transpose(1, 2))
    delta = torch.bmm(h * scale[at].reshape(streams, 1, 1), b[at].float().transpose(1, 2))
    y3 = y.float().reshape(delta.shape)
    return torch.where(has.reshape(streams, 1, 1), y3 + delta, y3).reshape(y.shape).to(y.dtype)


def _plain_verify(target, draft, tokens, u, lengths):
    B, K = tokens.shape
    p = target.double()
    P = p.sum(-1)
    p_tok = p[:, :K].gather(2, tokens.unsqueeze(-1)).squeeze(-1)
    if draft is None:                                              # the draft is sure of its token
        q_tok = Q = torch.ones_like(p_tok)
    else:
        Q = draft.double().sum(-1)
        q_tok = draft.gather(2, tokens.unsqueeze(-1)).squeeze(-1).double()
    step = torch.arange(K, device=tokens.device)
    n_draft = torch.full((B,), K, device=tokens.device) if lengths is None else lengths
    ok = (u[:, :K].double() * q_tok * P[:, :K] < p_tok * Q) & (step < n_draft.unsqueeze(-1))
    accepted = ok.long().cumprod(1).sum(1)
    rows, at = torch.arange(B, device=tokens.device), accepted.clamp(max=K - 1)
    pn = p[rows, accepted]
    if draft is None:
        left = pn.scatter(1, tokens[rows, at].unsqueeze(-1), 0.0)
    else:
        left = (pn * Q[rows, at].unsqueeze(-1) - draft[rows, at].double() * P[rows, at].unsqueeze(-1)).clamp(min=0.0)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, pn)
    w = torch.where((accepted < n_draft).unsqueeze(-1), left, pn)
    sums = w.cumsum(-1)
    hit = (w > 0) & (sums >= u[:, K:].double() * sums[:, -1:])
    place = torch.arange(w.shape[1], device=w.device)
    drawn = torch.where(hit.any(-1), hit.long().argmax(-1), torch.where(w > 0, place, -1).amax(-1))
    step = torch.arange(K + 1, device=tokens.device)
    padded = torch.cat([tokens, torch.full((B, 1), -1, device=tokens.device)], 1)
    n = accepted.unsqueeze(-1)
    return torch.where(step < n, padded, torch.where(step == n, drawn.unsqueeze(-1), -1)), accepted


def _plain_advance(state, counts, trace, params):
    L, _, B, T, C = trace.shape
    n = counts.reshape(B, 1, 1, 1)
    last = (counts - 1).clamp(min=0).reshape(1, 1, B, 1, 1).expand(L, 2, B, 1, C)
    x = trace[:, :2].gather(3, last).squeeze(3)                     # [L, 2, B, C]: the last accepted rows
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    carry = (x - mean) / torch.sqrt(var + EPS) * params[:, 0:3:2].unsqueeze(2) + params[:, 1:4:2].unsqueeze(2)
    k, v = trace[:, 2].transpose(0, 1), trace[:, 3].transpose(0, 1)  # [B, L, T, C]
    w = params[:, 4].unsqueeze(1)                                   # [L, 1, C]
    t = torch.arange(T, device=k.device).reshape(1, 1, T, 1)
    e = torch.where(t < n, k + (n - 1 - t) * w, -math.inf)
    e0 = state[:, :, 4].unsqueeze(2) + n * w                        # [B, L, 1, C]
    top = torch.maximum(e0, e.amax(2, keepdim=True))
    f, f0 = torch.exp(e - top), torch.exp(e0 - top)
    aa = f0 * state[:, :, 2].unsqueeze(2) + (f * v).sum(2, keepdim=True)
    bb = f0 * state[:, :, 3].unsqueeze(2) + f.sum(2, keepdim=True)
    new = torch.cat([carry.permute(2, 0, 1, 3), aa, bb, top], 2)
    return torch.where(n > 0, new, state)


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """Streams that have an adapter, and how many adapters those use."""
    with_one = case["streams"] - case["streams"] // 8
    return with_one, min(with_one, case["adapters"])


def work(case):
    if case["op"] == "adapt":
        k, outs = _site(case["embed"], case["site"])
        with_one, used = _pairs(case)
        rows, all_rows, r = with_one * case["tokens"], case["streams"] * case["tokens"], case["rank"]
        both = k * len(outs) + sum(outs)
        return {"bytes": used * r * both * ITEM[case["weights"]] + ITEM[case["rows"]] * (rows * k * len(outs) + 2 * all_rows * sum(outs)) + 8 * case["streams"],
                "flops": 2 * rows * r * both}
    if case["op"] == "verify":
        B, K, V = case["streams"], case["drafts"], case["vocab"]
        drafted = K / 2 if case["ragged"] else K                   # rows that may be needed; which are not depends on the numbers
        rows = B * (drafted + 1 + (drafted if case["draft_probs"] else 0))
        return {"bytes": 4 * rows * V + B * (8 * K + 4 * (K + 1) + 8 * (K + 1) + 8), "flops": 2 * rows * V}
    L, C, B, T = case["layers"], case["embed"], case["streams"], case["tokens"]
    n = (T + 1) / 2                                                # accepted tokens, on average
    return {"bytes": 4 * L * C * (B * (2 * n + 2 + 3 + 5) + 5) + 8 * B, "flops": L * C * B * (8 * n + 12)}


# ---------------------------------------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adapt":
        T, got = case["tokens"], []
        ids = s["ids"].tolist()
        for (a, b, scale), x, y in zip(s["banks"], s["xs"], s["ys"]):
            out = y.double()
            for i, j in enumerate(ids):
                if j >= 0:
                    h = x[i * T:(i + 1) * T].double() @ a[j].double().T
                    out[i * T:(i + 1) * T] += float(scale[j]) * (h @ b[j].double().T)
            got.append(out)
        return got
    if case["op"] == "verify":
        return _exact_verify(s)
    L, C, B, T = case["layers"], case["embed"], case["streams"], case["tokens"]
    out = s["state"].double()
    trace, w = s["trace"], s["params"].double()
    for i, n in enumerate(s["counts"].tolist()):
        if n == 0:
            continue
        for row, at in ((0, 0), (1, 2)):
            x = trace[:, row, i, n - 1].double()
            var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
            out[i, :, row] = w[:, at] * (x - mean) * (var + EPS).rsqrt() + w[:, at + 1]
        for t in range(n):
            k, v = trace[:, 2, i, t].double(), trace[:, 3, i, t].double()
            aa, bb, pp = out[i, :, 2].clone(), out[i, :, 3].clone(), out[i, :, 4] + w[:, 4]
            top = torch.maximum(pp, k)
            out[i, :, 2] = torch.exp(pp - top) * aa + torch.exp(k - top) * v
            out[i, :, 3] = torch.exp(pp - top) * bb + torch.exp(k - top)
            out[i, :, 4] = top
    return out


def _exact_verify(s):
    """Sequence by sequence and token by token on the host."""
    import numpy as np
    K = s["tokens"].shape[1]
    tokens, u = s["tokens"].cpu().numpy(), s["u"].cpu().numpy().astype(np.float64)
    lengths = None if s["lengths"] is None else s["lengths"].tolist()
    texts, counts = [], []
    for i in range(tokens.shape[0]):
        p = s["target"][i].cpu().numpy().astype(np.float64)
        q = None if s["draft"] is None else s["draft"][i].cpu().numpy().astype(np.float64)
        text, weights = [], None
        for t in range(K if lengths is None else lengths[i]):
            d = int(tokens[i, t])
            ps = p[t] / p[t].sum()
            qs = np.zeros_like(ps)
            if q is None:
                qs[d] = 1.0
            else:
                qs = q[t] / q[t].sum()
            if u[i, t] * qs[d] < ps[d]:
                text.append(d)
                continue
            weights = np.maximum(ps - qs, 0.0)
            if not weights.sum() > 0:
                weights = ps
            break
        if weights is None:
            weights = p[len(text)]
        sums = np.cumsum(weights)
        hits = np.nonzero((weights > 0) & (sums >= u[i, K] * sums[-1]))[0]
        counts.append(len(text))
        text.append(int(hits[0]) if hits.size else int(np.nonzero(weights > 0)[0][-1]))
        texts.append(text + [-1] * (K + 1 - len(text)))
    return torch.tensor(texts), torch.tensor(counts)
