"""Plain definitions, in 64 bits on the CPU, of the operators over a vocabulary,
inputs for them and the tolerances that their arithmetic allows."""
import math

import torch

INF = math.inf


def log_softmax(x, temperature):
    """Rows of log p in 64 bits; a row of nothing but -inf has -inf throughout."""
    z = x.double() / temperature
    m = z.amax(-1, keepdim=True)
    t = z - torch.where(m == -INF, torch.zeros_like(m), m)
    s = torch.exp(t).sum(-1, keepdim=True)
    return torch.where(s == 0, torch.full_like(t, -INF), t - torch.log(s))


def token_scores(logits, tokens, top_k, temperature=1.0, ignore_index=-100):
    """(log_probs, entropy, top_tokens, top_log_probs) of logits [R, V], tokens [R]."""
    logits, tokens = logits.detach().cpu(), tokens.detach().cpu().long()
    logp = log_softmax(logits, temperature)
    p = torch.exp(logp)
    h = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(1)
    v = logits.shape[1]
    skip, bad = tokens == ignore_index, (tokens < 0) | (tokens >= v)
    lp = logp.gather(1, tokens.clamp(0, v - 1)[:, None])[:, 0]
    lp = torch.where(bad, torch.full_like(lp, math.nan), lp)
    top = torch.sort(logits.float(), dim=1, descending=True, stable=True).indices[:, :top_k]
    tlp = logp.gather(1, top)
    lp, h = lp.masked_fill(skip, 0.0), h.masked_fill(skip, 0.0)
    return lp, h, top.masked_fill(skip[:, None], -1), tlp.masked_fill(skip[:, None], 0.0)


def token_scores_grad(logits, tokens, g_lp, g_h, temperature=1.0, ignore_index=-100):
    """Gradient of the logits from the formula."""
    logits, tokens = logits.detach().cpu(), tokens.detach().cpu().long()
    v = logits.shape[1]
    logp = log_softmax(logits, temperature)
    p = torch.exp(logp)
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    h = -plogp.sum(1, keepdim=True)
    gl, gh = g_lp.detach().cpu().double()[:, None], g_h.detach().cpu().double()[:, None]
    dx = -gl * p - gh * (plogp + p * h)
    dx.scatter_add_(1, tokens.clamp(0, v - 1)[:, None], gl)
    dx[(tokens < 0) | (tokens >= v)] = math.nan
    dx[(logits == -INF).all(1)] = 0.0
    dx[tokens == ignore_index] = 0.0
    return dx / temperature


def distill(logits, teacher_tokens, teacher_logits, temperature=1.0, weight=1.0):
    """(loss of each row, rows that have a teacher, gradient of the sum of the row losses)."""
    logits, tok = logits.detach().cpu(), teacher_tokens.detach().cpu().long()
    v = logits.shape[1]
    z = torch.where(tok < 0, torch.full(tok.shape, -INF, dtype=torch.float64), teacher_logits.detach().cpu().double())
    some = (z != -INF).any(1)
    logq = log_softmax(z, temperature)
    q = torch.exp(logq)
    logp = log_softmax(logits, temperature)
    at = tok.clamp(0, v - 1)
    term = torch.where(q == 0, torch.zeros_like(q), q * (logq - logp.gather(1, at)))
    scale = weight * temperature * temperature
    loss = scale * term.sum(1)
    dx = torch.exp(logp).scatter_add_(1, at, -q) * (weight * temperature)
    dx[(logits == -INF).all(1)] = 0.0
    bad = (tok >= v).any(1)
    loss[bad] = math.nan
    dx[bad] = math.nan
    loss[~some] = 0.0
    dx[~some] = 0.0
    return loss, some, dx


def embedding_grad(tokens, dy, vocab, scale, padding_idx=None):
    tokens = tokens.detach().cpu().long().reshape(-1)
    dy = dy.detach().cpu().double().reshape(tokens.numel(), -1)
    ok = (tokens >= 0) & (tokens < vocab)
    dw = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    dw.index_add_(0, tokens[ok], dy[ok])
    if padding_idx is not None:
        dw[padding_idx] = 0.0
    return dw * scale


# What one rounding to a type changes, relative and (below its normal numbers) absolute.
ROUNDING = {torch.float32: (2.0 ** -24, 2.0 ** -149), torch.bfloat16: (2.0 ** -9, 2.0 ** -134),
            torch.float16: (2.0 ** -11, 2.0 ** -25)}


def spread(logits, temperature):
    """Largest distance of a finite logit from its row's largest that still matters
    to the sums (2^-24 of the largest probability and below do not), over T."""
    x = logits.detach().cpu().double()
    x = x[torch.isfinite(x)]
    if x.numel() == 0:
        return 1.0
    return max(1.0, min(float(x.max() - x.min()) / temperature, 200.0))


def score_tolerance(logits, temperature):
    """Absolute error of a log probability or an entropy in fp32 arithmetic.  A
    value's exponent carries 3 roundings of 2^-24 relative (difference, scaling,
    constant); the exponential and the sums (of at most 256 terms in a row, then
    trees) add 2^-23 and 2^-24 * 256 / 2 at worst; values far from the largest
    enter by their share.  The log probability itself is rounded at its size."""
    return 2.0 ** -24 * (6 * spread(logits, temperature) + 150)


def assert_close(name, got, ref, dtype, atol):
    """got (dtype) against ref (64 bits): within atol and the type's rounding (up to
    two units where the value sits at a boundary), infinities and NaN in the same places."""
    got, ref = got.detach().cpu().double(), ref.cpu().double()
    # (what rounds past the type's range is infinite in it)
    ref = torch.where(torch.isinf(ref.to(dtype)), ref.to(dtype).double(), ref)
    assert got.shape == ref.shape, (name, got.shape, ref.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN in other places"
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]) and torch.equal(torch.isinf(got), inf), f"{name}: other infinities"
    ok = torch.isfinite(ref)
    if not ok.any():
        return
    rel, tiny = ROUNDING[dtype]
    err = (got[ok] - ref[ok]).abs() - (2 * rel * ref[ok].abs() + tiny + atol)
    assert err.max().item() <= 0.0, f"{name}: beyond the tolerance by {err.max().item():.3e} (atol {atol:.3e})"
