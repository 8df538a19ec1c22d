"""The operators over a vocabulary whose speed is measured: log probabilities of
given tokens with entropy and top alternatives, distillation from a teacher's
top logits, and the scaled token embedding, each with its gradient.

A case is a dict of plain values:

  op           "log_probs" (no gradient), "log_probs_train", "distill", "embed" (no gradient), "embed_train"
  rows         positions (tokens of all texts of a call)
  vocab        size of the vocabulary
  dtype        "f32", "bf16", "f16": element type of the logits or of the embedding's weight
  k            top alternatives asked for, or entries of the teacher per position
  temperature  of the softmax
  pad          share of the positions that are padding
  stride       elements between the rows of the logits (0: rows follow one another)
  loss_scale   the gradient that the loss gets in the backward pass (programs in fp16 scale their losses)
  dim          features of the embedding

With ``own`` false every operator is computed in its plain form, in elementary
torch operations in 32 bits, rounded once at the end; with ``own`` true by this
package.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORE = -100


def _scores(name, op, rows, vocab, dtype, k=0, temperature=1.0, pad=0.0, stride=0):
    c = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype, "k": k, "temperature": temperature, "pad": pad,
         "stride": stride}
    if op == "distill":
        c["loss_scale"] = 1024.0 if dtype == "f16" else 1.0
    return {"name": name, **c} if name else c


def _embed(name, op, rows, vocab, dim, dtype, pad=0.0):
    c = {"op": op, "rows": rows, "vocab": vocab, "dim": dim, "dtype": dtype, "pad": pad}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one token of one text being generated, with the alternatives an interface shows: latency
        _scores("log_probs_bf16_1x131072_top20", "log_probs", 1, 131072, "bf16", k=20),
        # a batch of texts being generated; a vocabulary that no vector width divides, fp32 logits
        _scores("log_probs_f32_48x50001_top5", "log_probs", 48, 50001, "f32", k=5, temperature=0.7),
        # a teacher scores a batch and hands on its top logits
        _scores("log_probs_bf16_4096x131072_top32", "log_probs", 4096, 131072, "bf16", k=32, temperature=2.0, pad=0.1),
        # captions' log probabilities and entropy as a training signal
        _scores("log_probs_train_bf16_8192x49408", "log_probs_train", 8192, 49408, "bf16", pad=0.25),
        # a small debugging batch, and a column slice of a padded logits matrix in fp16
        _scores("distill_f32_64x8192_top8", "distill", 64, 8192, "f32", k=8, temperature=2.0),
        _scores("distill_f16_1003x32001_top10", "distill", 1003, 32001, "f16", k=10, temperature=1.5, pad=0.2,
                stride=32064),
        # a student trained on the captions of a batch
        _scores("distill_bf16_8192x49408_top32", "distill", 8192, 49408, "bf16", k=32, temperature=2.0, pad=0.25),
        # the largest vocabulary
        _scores("distill_bf16_4096x200000_top64", "distill", 4096, 200000, "bf16", k=64),
        # the next token's features while a text is generated
        _embed("embed_bf16_32x49408x768", "embed", 32, 49408, 768, "bf16"),
        # sizes that no vector width divides, fp32
        _embed("embed_train_f32_5003x32001x641", "embed_train", 5003, 32001, 641, "f32", pad=0.2),
        # the texts of a contrastive batch: 1024 of 77 tokens, nearly half of them padding
        _embed("embed_train_bf16_78848x49408x768", "embed_train", 78848, 49408, 768, "bf16", pad=0.45),
        # the largest batch of tokens
        _embed("embed_train_bf16_524288x131072x1024", "embed_train", 524288, 131072, 1024, "bf16", pad=0.1),
    ]


# no drawn case moves more bytes than the largest listed one
_MOST_BYTES = 3.2e9


def _log_uniform(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    op = rng.choice(["log_probs", "log_probs", "log_probs_train", "distill", "distill", "embed", "embed_train",
                     "embed_train"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    while True:
        # vocabularies: mostly whole vectors, now and then any size
        vocab = _log_uniform(rng, 1000, 200000)
        q = rng.choice([64, 64, 8, 1])
        vocab = max(q, vocab // q * q)
        pad = rng.choice([0.0, 0.1, 0.45])
        if op.startswith("embed"):
            rows = _log_uniform(rng, 1, 524288)
            dim = _log_uniform(rng, 64, 1536)
            q = rng.choice([64, 64, 8, 1])
            c = _embed(None, op, rows, vocab, max(q, dim // q * q), dtype, pad=pad)
        else:
            k = rng.choice([1, 5, 10, 20, 32, 64])
            if op == "log_probs":
                k = rng.choice([0, k])
            elif op == "log_probs_train":
                k = 0
            stride = rng.choice([0, 0, (vocab + 127) // 64 * 64])
            c = _scores(None, op, _log_uniform(rng, 1, 16384), vocab, dtype, k=k,
                        temperature=rng.choice([0.7, 1.0, 1.0, 2.0]), pad=pad, stride=stride)
        if work(c)["bytes"] < _MOST_BYTES:
            return c


def _randn(shape, g):
    return torch.randn(shape, generator=g, device="cuda")


def _tokens(n, vocab, g):
    """Tokens as texts have them: frequencies fall off like 1 / rank, over all of the vocabulary."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    rank = (torch.exp(u * math.log(vocab)) - 1.0).long().clamp_(0, vocab - 1)
    return (rank * 7919 + 13) % vocab if math.gcd(7919, vocab) == 1 else rank


def _padded(n, share, g):
    return torch.rand(n, generator=g, device="cuda") < share


def _logits(case, g):
    """A model's logits: a wide bulk and some tokens that stand out of it."""
    rows, vocab, stride = case["rows"], case["vocab"], case["stride"] or case["vocab"]
    dtype = _DTYPES[case["dtype"]]
    x = torch.empty((rows, stride), device="cuda", dtype=dtype)
    step = max(1, (1 << 28) // stride)
    for i in range(0, rows, step):
        n = min(step, rows - i)
        z = _randn((n, stride), g).mul_(2.0)
        at = torch.randint(0, vocab, (n, 12), generator=g, device="cuda")
        z.scatter_add_(1, at, 6.0 + 2.0 * _randn((n, 12), g))
        x[i:i + n] = z.to(dtype)
    return x[:, :vocab]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, vocab = case["op"], case["rows"], case["vocab"]
    state = {"case": case}
    if op.startswith("embed"):
        dtype = _DTYPES[case["dtype"]]
        weight = _randn((vocab, case["dim"]), g).div_(math.sqrt(case["dim"])).to(dtype)
        tokens = _tokens(rows, vocab, g)
        # padding is a token of its own here, the last one, and has no gradient
        tokens[_padded(rows, case["pad"], g)] = vocab - 1
        train = op == "embed_train"
        state.update(tokens=tokens, weight=weight.requires_grad_(train), scale=math.sqrt(case["dim"]),
                     padding=vocab - 1)
        if train:
            state["dy"] = _randn((rows, case["dim"]), g).div_(16.0).to(dtype)
        return state
    x = _logits(case, g)
    padded = _padded(rows, case["pad"], g)
    state["logits"] = x.requires_grad_(op != "log_probs")
    if op == "distill":
        k = case["k"]
        # a teacher's tokens in the order of its log probabilities, no token twice in a row
        first = torch.randint(0, vocab, (rows, 1), generator=g, device="cuda")
        hop = torch.randint(1, max(2, vocab // k), (rows, 1), generator=g, device="cuda")
        tokens = (first + hop * torch.arange(k, device="cuda")) % vocab
        tokens[padded] = -1
        lp = torch.sort(torch.log_softmax(_randn((rows, k), g).mul_(2.0), 1), dim=1, descending=True).values - 0.2
        state.update(teacher_tokens=tokens, teacher_logits=lp,
                     g_loss=torch.full((), case["loss_scale"], device="cuda"))
    else:
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        tokens[padded] = _IGNORE
        state["tokens"] = tokens
        if op == "log_probs_train":
            # an advantage for each token, and an entropy bonus
            state["g_log_probs"] = -_randn((rows,), g) / rows
            state["g_entropy"] = torch.full((rows,), -0.01 / rows, device="cuda")
    return state


# ---- plain forms ----


def _plain_softmax(x, temperature):
    """t = z - max z, log of the sum, probabilities; a row of nothing but -inf has no probability anywhere."""
    z = x / temperature
    m = z.amax(1, keepdim=True)
    t = z - torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(t)
    s = e.sum(1, keepdim=True)
    return t, torch.log(s), e / torch.where(s == 0, torch.ones_like(s), s)


def _plain_log_probs(s):
    c = s["case"]
    x, tokens, k, temperature = s["logits"].detach(), s["tokens"], c["k"], c["temperature"]
    skip = tokens == _IGNORE
    xf = x.float()
    t, ls, p = _plain_softmax(xf, temperature)
    zero = torch.zeros((), device=x.device)
    at = tokens.clamp_min(0)[:, None]
    lp = torch.where(skip, zero, (t.gather(1, at) - ls)[:, 0])
    logp = t - ls
    plogp = torch.where(p > 0, p * logp, zero)
    h = torch.where(skip, zero, -plogp.sum(1))
    out = {"log_probs": lp, "entropy": h}
    if c["op"] == "log_probs_train":
        gl = torch.where(skip, zero, s["g_log_probs"])[:, None]
        gh = torch.where(skip, zero, s["g_entropy"])[:, None]
        dx = -(gl * p) - gh * (plogp + p * h[:, None])
        dx.scatter_add_(1, at, gl)
        out["dx"] = (dx / temperature).to(x.dtype)
    elif k:
        top = torch.sort(xf, dim=1, descending=True, stable=True).indices[:, :k].contiguous()
        out["top_tokens"] = torch.where(skip[:, None], -torch.ones_like(top), top)
        out["top_log_probs"] = torch.where(skip[:, None], zero, t.gather(1, top) - ls)
    return out


def _plain_distill(s):
    c = s["case"]
    x, tokens, temperature = s["logits"].detach(), s["teacher_tokens"], c["temperature"]
    t, ls, p = _plain_softmax(x.float(), temperature)
    valid = tokens >= 0
    some = valid.any(1)
    zero = torch.zeros((), device=x.device)
    z = torch.where(valid, s["teacher_logits"].float() / temperature, zero - math.inf)
    tq, lsq, q = _plain_softmax(z, 1.0)
    at = tokens.clamp_min(0)
    term = torch.where(q > 0, q * ((tq - lsq) - (t.gather(1, at) - ls)), zero)
    n = some.sum().clamp_min(1)
    loss = temperature * temperature * term.sum() / n
    dx = p.mul_(some[:, None]).scatter_add_(1, at, -q)
    return {"loss": loss, "dx": (dx * (s["g_loss"] * temperature / n)).to(x.dtype)}


def _plain_embed(s):
    w, tokens = s["weight"].detach(), s["tokens"]
    out = {"y": (w[tokens].float() * s["scale"]).to(w.dtype)}
    if s["case"]["op"] == "embed_train":
        dw = torch.zeros(w.shape, device=w.device)
        dw.index_add_(0, tokens, s["dy"].float())
        dw[s["padding"]] = 0.0
        out["dweight"] = (dw * s["scale"]).to(w.dtype)
    return out


# ---- the framework's operators ----


def _own(s):
    import memoryefficientclip_amd as mec

    c = s["case"]
    if c["op"].startswith("embed"):
        w = s["weight"]
        if c["op"] == "embed":
            with torch.no_grad():
                return {"y": mec.scaled_embedding(s["tokens"], w, s["scale"], padding_idx=s["padding"])}
        w.grad = None
        y = mec.scaled_embedding(s["tokens"], w, s["scale"], padding_idx=s["padding"])
        y.backward(s["dy"])
        return {"y": y.detach(), "dweight": w.grad}
    x = s["logits"]
    if c["op"] == "log_probs":
        with torch.no_grad():
            r = mec.token_log_probs(x, s["tokens"], top_k=c["k"], temperature=c["temperature"])
        out = {"log_probs": r.log_probs, "entropy": r.entropy}
        if c["k"]:
            out["top_tokens"], out["top_log_probs"] = r.top_tokens, r.top_log_probs
        return out
    x.grad = None
    if c["op"] == "log_probs_train":
        r = mec.token_log_probs(x, s["tokens"], temperature=c["temperature"])
        torch.autograd.backward([r.log_probs, r.entropy], [s["g_log_probs"], s["g_entropy"]])
        return {"log_probs": r.log_probs.detach(), "entropy": r.entropy.detach(), "dx": x.grad}
    loss = mec.TopKDistillationLoss(temperature=c["temperature"])(x, s["teacher_tokens"], s["teacher_logits"])
    loss.backward(s["g_loss"])
    return {"loss": loss.detach(), "dx": x.grad}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op.startswith("embed"):
        return _plain_embed(state)
    return _plain_distill(state) if op == "distill" else _plain_log_probs(state)


def work(case):
    """Each input read once and each output written once; rows of logits that are padding need no read."""
    rows, vocab, size, op = case["rows"], case["vocab"], _SIZE[case["dtype"]], case["op"]
    if op.startswith("embed"):
        dim = case["dim"]
        # the gathered rows, at most one read of the whole weight
        n = 8.0 * rows + (min(rows, vocab) + rows) * dim * size
        f = 1.0 * rows * dim
        if op == "embed_train":
            n += (rows * (1.0 - case["pad"]) + vocab) * dim * size
            f += (rows + vocab) * dim
        return {"bytes": n, "flops": f}
    live = rows * (1.0 - case["pad"])
    if op == "distill":
        return {"bytes": (live + rows) * vocab * size + 12.0 * rows * case["k"] + 4, "flops": 7.0 * live * vocab}
    n = live * vocab * size + rows * (16.0 + 12.0 * case["k"])
    f = 6.0 * live * vocab
    if op == "log_probs_train":
        n += rows * (vocab * size + 8.0)
        f += 6.0 * live * vocab
    return {"bytes": n, "flops": f}


# ---- the definitions in 64 bits ----


def _exact_distribution(x, temperature):
    """log p and p of rows x in 64 bits."""
    z = x.double() / temperature
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    return logp, torch.exp(logp)


def exact(case, seed):
    s = prepare(case, seed)
    op, rows, vocab = case["op"], case["rows"], case["vocab"]
    if op.startswith("embed"):
        w = s["weight"].detach().double()
        out = {"y": w[s["tokens"]] * s["scale"]}
        if op == "embed_train":
            keep = s["tokens"] != s["padding"]
            order = torch.argsort(s["tokens"][keep], stable=True)
            dy = s["dy"][keep][order].double()
            count = torch.bincount(s["tokens"][keep], minlength=vocab)
            # sums of runs as differences of running sums, in 64 bits
            run = torch.cat([torch.zeros_like(dy[:1]), dy.cumsum(0)]) if dy.shape[0] else dy.new_zeros((1, case["dim"]))
            end = count.cumsum(0)
            out["dweight"] = (run[end] - run[end - count]) * s["scale"]
        return out
    x, t = s["logits"].detach(), case["temperature"]
    parts = []
    if op == "distill":
        tokens = s["teacher_tokens"]
        some = (tokens >= 0).any(1)
        n = max(1, int(some.sum()))
    step = max(1, (1 << 27) // vocab)
    for i in range(0, rows, step):
        at = slice(i, min(rows, i + step))
        logp, p = _exact_distribution(x[at], t)
        if op == "distill":
            tok, live = tokens[at].clamp_min(0), some[at, None].double()
            logq, q = _exact_distribution(s["teacher_logits"][at], t)
            loss = (live * q * (logq - logp.gather(1, tok))).sum() * (t * t / n)
            dx = (live * p).scatter_add_(1, tok, -live * q) * (case["loss_scale"] * t / n)
            parts.append((loss, dx))
            continue
        tok = s["tokens"][at]
        live = tok != _IGNORE
        tok = tok.clamp_min(0)[:, None]
        lp = logp.gather(1, tok)[:, 0] * live
        h = -torch.xlogy(p, p).sum(1) * live
        if op == "log_probs_train":
            gl = (s["g_log_probs"][at].double() * live)[:, None]
            gh = (s["g_entropy"][at].double() * live)[:, None]
            dx = -p * (gl + gh * (logp + h[:, None]))
            dx.scatter_add_(1, tok, gl)
            parts.append((lp, h, dx / t))
        elif case["k"]:
            top = torch.sort(x[at].float(), dim=1, descending=True, stable=True).indices[:, :case["k"]]
            tlp = logp.gather(1, top) * live[:, None]
            parts.append((lp, h, torch.where(live[:, None], top, -torch.ones_like(top)), tlp))
        else:
            parts.append((lp, h))
    if op == "distill":
        return {"loss": sum(q[0] for q in parts), "dx": torch.cat([q[1] for q in parts])}
    names = ["log_probs", "entropy", "dx"] if op == "log_probs_train" else ["log_probs", "entropy", "top_tokens",
                                                                            "top_log_probs"]
    return {k: torch.cat(v) for k, v in zip(names, zip(*parts))}
