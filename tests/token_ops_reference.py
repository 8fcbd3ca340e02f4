"""Token log probabilities, embeddings and their gradients in 64 bits on the
CPU, straight from their formulas, with bounds for what fp32 arithmetic may
differ by: U = 2^-24 is half a step of fp32, HALF[t] of the output's type."""
import torch

U = 2.0 ** -24
HALF = {torch.bfloat16: torch.finfo(torch.bfloat16).eps / 2, torch.float32: U}
IGNORE = -100
NAN, INF = float("nan"), float("inf")


def token_logprobs(logits, tokens, scale=1.0, ignore_index=IGNORE, top=0):
    """(logprob, lse, entropy, top values, top ids) and their tolerances."""
    rows, vocab = logits.shape
    x = logits.double().cpu()
    s = x * float(torch.tensor(scale, dtype=torch.float32))
    m = s.max(-1).values
    special = ~torch.isfinite(m)
    t = s - m[:, None]
    e = torch.exp(t)
    z = e.sum(-1)
    log_z = torch.log(z)
    at = torch.where(e > 0, t.abs(), 0.0)
    mean_t, mean_t2 = (e * at).sum(-1) / z, (e * at * at).sum(-1) / z
    lse = torch.where(special, torch.where(torch.isnan(x).any(-1), torch.tensor(NAN).double(), m),
                      m + log_z)
    entropy = torch.where(special, torch.tensor(NAN).double(), log_z + mean_t)
    toks = tokens.long().cpu()
    skip = toks == ignore_index
    known = (toks >= 0) & (toks < vocab)
    at_token = s.gather(1, torch.where(known, toks, 0)[:, None])[:, 0]
    # s - lse, where lse = m + ln Z may hide ln Z behind a huge m.
    minus_lse = lambda v: torch.where(special, v - lse, (v - m) - log_z)  # noqa: E731
    logprob = torch.where(known, minus_lse(at_token), torch.tensor(NAN).double())
    # A sum of `adds` terms in a row is off by at most `adds` halves of a step,
    # each term by 3 (its difference, product and exp2 argument, times |t|)
    # and 2 for exp2; a rescaling of the sums costs 4 more, at most 32 deep.
    adds = vocab / 64 + 64 + 128
    tol_z = U * (3 * mean_t + adds)
    tol_lse = tol_z + U * (2 * m.abs() + 2 * lse.abs() + 4 * log_z.abs())
    tol_lp = tol_z + U * (4 * (at_token - m).abs() + 2 * logprob.abs() + 4 * log_z.abs())
    tol_h = (tol_z * (1 + mean_t) + U * (3 * mean_t2 + adds * mean_t + 8 * mean_t
                                         + 4 * log_z.abs() + 2 * entropy.abs()))
    zero = torch.zeros((), dtype=torch.float64)
    # NaN counts as the largest, equal values keep their order.
    order = torch.sort(x, dim=-1, descending=True, stable=True)
    ids = order.indices[:, :top]
    st = s.gather(1, ids)
    values = torch.stack([minus_lse(v) for v in st.unbind(1)], 1) if top else st
    tol_top = tol_z[:, None] + U * (4 * (st - m[:, None]).abs() + 2 * values.abs()
                                    + 4 * log_z.abs()[:, None])
    logprob, lse, entropy = (torch.where(skip, zero, v) for v in (logprob, lse, entropy))
    values = torch.where(skip[:, None], torch.tensor(-INF).double(), values)
    ids = torch.where(skip[:, None], -1, ids)
    logprob, lse, values = (fp32_range(v) for v in (logprob, lse, values))
    return (logprob, lse, entropy, values, ids), (tol_lp, tol_lse, tol_h, tol_top)


def fp32_range(v):
    """What fp32 rounds to infinity is infinite."""
    return torch.where(torch.isfinite(v) & torch.isinf(v.float()), v.float().double(), v)


def token_logprobs_bwd(grad, logits, tokens, lse, scale=1.0, ignore_index=IGNORE, entropy=None,
                       grad_entropy=None, grad_lse=None):
    """dlogits in 64 bits from the same lse and entropy, and its tolerance."""
    rows, vocab = logits.shape
    out_half = HALF[logits.dtype]
    d64 = lambda v: torch.zeros(rows, 1).double() if v is None else v.double().cpu()[:, None]  # noqa: E731
    scale = float(torch.tensor(scale, dtype=torch.float32))
    x = logits.double().cpu() * scale
    g, gh, gl, h = d64(grad), d64(grad_entropy), d64(grad_lse), d64(entropy)
    lp = x - d64(lse)
    p = torch.exp(lp)
    lp0 = torch.where(p > 0, lp, 0.0)
    inner = gl - g - gh * (lp0 + h)
    toks = tokens.long().cpu()[:, None]
    hot = (torch.arange(vocab)[None] == toks).double()
    d = hot * g + p * inner
    # ln p: one rounding (of |ln p|); p: that times p, and 4 for the exponential;
    # the bracket: 2 products and 3 sums of its parts; the last sum and product 2.
    size = gl.abs() + g.abs() + gh.abs() * (lp0.abs() + h.abs())
    tol = scale * U * (p * size * (lp0.abs() + 12) + 3 * d.abs())
    # Below 2^-126 a product may be flushed, and p under e^-87 likewise.
    tol = tol + scale * 2.0 ** -125 * (1 + size)
    dx = scale * d
    tol = tol + out_half * dx.abs() * (1 + 2.0 ** -10) + 2.0 ** -133
    known = (toks >= 0) & (toks < vocab)
    dx = torch.where(known, dx, torch.tensor(NAN).double())
    return torch.where(toks == ignore_index, torch.zeros((), dtype=torch.float64), dx), tol


def embedding(weight, tokens, scale=1.0):
    scale = float(torch.tensor(scale, dtype=torch.float32))
    toks = tokens.long().cpu()
    known = (toks >= 0) & (toks < weight.shape[0])
    w = weight.double().cpu()[torch.where(known, toks, 0)] * scale
    return torch.where(known[..., None], w, torch.tensor(NAN).double())


def embedding_bwd(grad, tokens, vocab, scale=1.0, padding_idx=None, into=None,
                  dtype=torch.float32):
    """dweight in 64 bits and its tolerance."""
    scale = float(torch.tensor(scale, dtype=torch.float32))
    width = grad.shape[-1]
    g = grad.double().cpu().reshape(-1, width)
    toks = tokens.long().cpu().reshape(-1)
    use = (toks >= 0) & (toks < vocab)
    if padding_idx is not None:
        use &= toks != padding_idx
    g, toks = g[use], toks[use]
    dw = torch.zeros(vocab, width, dtype=torch.float64)
    size = torch.zeros(vocab, width, dtype=torch.float64)
    dw.index_add_(0, toks, g)
    size.index_add_(0, toks, g.abs())
    n = torch.bincount(toks, minlength=vocab).double()[:, None]
    out = dw * scale + (0 if into is None else into.double().cpu())
    # A sum of n terms in any order: n - 1 halves of a step of the sum of their
    # absolute values; the product and the sum with `into` one each.
    tol = U * (n * size * abs(scale) + out.abs() + (dw * scale).abs())
    tol = tol + HALF[dtype] * out.abs() * (1 + 2.0 ** -10) + 2.0 ** -133
    touched = (n > 0)[:, 0]
    return out, tol, touched


def close(got, want, tol, what):
    """NaN and infinities in the same places, the others within tol."""
    got = got.detach().double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), \
        f"{what}: infinities in other places"
    tol = torch.where(torch.isnan(tol), 0.0, tol)  # of a row that is left out: exact
    over = ((got - want).abs() - tol)[fine]
    assert not over.numel() or float(over.max()) <= 0, (
        f"{what}: off by {float((got - want).abs()[fine].max()):.3e}, "
        f"{float(over.max()):.3e} over the bound")
