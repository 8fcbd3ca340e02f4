"""The norms around a block and the output layer's cross entropy, with their
gradients, in 64 bits straight from their formulas, with bounds for what fp32
arithmetic may differ by: U = 2^-24 is half a step of fp32, HALF[t] of the
output's type.  A value's bound stands beside it, as "tol"."""
import torch

from token_ops_reference import HALF, IGNORE, INF, NAN, U, close  # noqa: F401

BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64

# Additions that one value passes through in a row's sum: 16 of a lane, 6 of a
# wave, 16 of the waves; with the products and the division by the width.
ROW_ADDS = 48


def f32(v):
    """A number as the kernels get it."""
    return float(torch.tensor(v, dtype=F32))


def rounded(value, tol, dtype):
    """The bound after the one rounding to dtype."""
    return tol + HALF[dtype] * (value.abs() + tol) + 2.0 ** -133


def _norm(v, weight, bias, layer, offset, eps):
    """y, its bound, and (mean, rstd) with theirs, of rows that are exact."""
    mean = v.mean(-1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    tol_mean = U * ROW_ADDS * v.abs().mean(-1, keepdim=True) if layer else mean
    c = v - mean
    tol_c = tol_mean + U * c.abs()
    var = c.square().mean(-1, keepdim=True)
    tol_var = 2 * (c.abs() * tol_c).mean(-1, keepdim=True) + tol_c.square().mean(
        -1, keepdim=True) + U * ROW_ADDS * var
    rstd = (var + eps).rsqrt()
    # The root and the quotient are off by a step each at most.
    tol_rstd = rstd * (0.5 * tol_var / (var + eps) + 6 * U)
    w = weight + offset
    e = c * rstd
    tol_e = tol_c * rstd + c.abs() * tol_rstd + 2 * U * e.abs()
    y = e * w + (0 if bias is None else bias)
    tol_y = tol_e * w.abs() + 3 * U * (e * w).abs() + U * y.abs()
    return y, tol_y, (mean, rstd), (tol_mean, tol_rstd)


def _rows_of_gate(gate, rows, like):
    if gate is None:
        return torch.ones(1, 1, dtype=F64, device=like.device)
    g = gate.double().reshape(-1, like.shape[1])
    return g.repeat_interleave(rows // g.shape[0], 0)


def _opt(t):
    return None if t is None else t.double()


def stream(x, residual, *, post=None, post_bias=None, gate=None, norm="rms", scale=1.0,
           offset=0.0, eps=1e-6, **_):
    """h and the statistics of x, with their bounds."""
    n, tol_n = x.double(), torch.zeros_like(x, dtype=F64)
    one = torch.ones(x.shape[0], 1, dtype=F64, device=x.device)
    stats, tol_stats = (0 * one, one), (0 * one, 0 * one)
    if post is not None:
        n, tol_n, stats, tol_stats = _norm(n, post.double(), _opt(post_bias), norm == "layer",
                                           f32(offset), f32(eps))
    g = _rows_of_gate(gate, x.shape[0], x) * f32(scale)
    h = residual.double() + n * g
    tol = tol_n * g.abs() + 2 * U * (n * g).abs() + U * h.abs()
    return h, rounded(h, tol, x.dtype), torch.cat(stats, -1), torch.cat(tol_stats, -1)


def after(h, *, pre=None, pre_bias=None, norm="rms", offset=0.0, eps=1e-6, **_):
    """y and the statistics of h as it is stored, with their bounds."""
    y, tol, stats, tol_stats = _norm(h.double(), pre.double(), _opt(pre_bias), norm == "layer",
                                     f32(offset), f32(eps))
    return y, rounded(y, tol, h.dtype), torch.cat(stats, -1), torch.cat(tol_stats, -1)


def _norm_bwd(g, tol_g, v, mean, rstd, weight, layer):
    """Of the rows, the weight and the bias: [(gradient, bound)]."""
    e = (v - mean) * rstd
    tol_e = 2 * U * rstd.abs() * (v.abs() + mean.abs()) + U * e.abs()
    u = g * weight
    tol_u = tol_g * weight.abs() + 2 * U * u.abs()
    ue = u * e
    tol_ue = tol_u * e.abs() + u.abs() * tol_e + U * ue.abs()
    mean_of = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    m = mean_of(ue)
    tol_m = mean_of(tol_ue) + U * ROW_ADDS * mean_of(ue.abs())
    mu = mean_of(u) if layer else 0 * m
    tol_mu = mean_of(tol_u) + U * ROW_ADDS * mean_of(u.abs()) if layer else 0 * m
    d = rstd * (u - e * m - mu)
    tol_d = rstd.abs() * (tol_u + e.abs() * tol_m + tol_e * m.abs() + tol_mu
                          + 4 * U * (u.abs() + (e * m).abs() + mu.abs()))
    # Sums over rows: as many additions as rows at most.
    ge = g * e
    adds = U * (g.shape[0] + 2)
    dw = ge.sum(0), (tol_g * e.abs() + g.abs() * tol_e).sum(0) + adds * ge.abs().sum(0)
    db = g.sum(0), tol_g.sum(0) + adds * g.abs().sum(0)
    return (d, tol_d), dw, db


def block_norms_bwd(grad_h, grad_y, x, h, stats, *, post=None, post_bias=None, pre=None,
                    pre_bias=None, gate=None, norm="rms", scale=1.0, offset=0.0):
    """[(gradient, bound) or None] in the order of the library's results."""
    layer, offset, scale = norm == "layer", f32(offset), f32(scale)
    rows, cols = x.shape
    st = stats.double()[:, :, None]
    total = torch.zeros_like(x, dtype=F64) if grad_h is None else grad_h.double()
    tol = torch.zeros_like(total)
    dpre = dpre_bias = dgate = dpost = dpost_bias = None
    if pre is not None:
        gy = grad_y.double()
        (d, tol_d), dpre, dpre_bias = _norm_bwd(gy, torch.zeros_like(gy), h.double(), st[:, 2],
                                                st[:, 3], pre.double() + offset, layer)
        total = total + d
        tol = tol_d + U * total.abs()
    g = _rows_of_gate(gate, rows, x) * scale
    xd = x.double()
    if gate is not None:
        n, tol_n = xd, torch.zeros_like(xd)
        if post is not None:
            w = post.double() + offset
            e = (xd - st[:, 0]) * st[:, 1]
            n = e * w + (0 if post_bias is None else post_bias.double())
            tol_n = (2 * U * st[:, 1].abs() * (xd.abs() + st[:, 0].abs()) + 3 * U * e.abs()
                     ) * w.abs() + U * n.abs()
        tn = total * n * scale
        tol_tn = (tol * n.abs() + total.abs() * tol_n) * abs(scale) + 3 * U * tn.abs()
        shape = (gate.numel() // cols, -1, cols)
        dgate = tn.reshape(shape).sum(1), tol_tn.reshape(shape).sum(1) + U * (
            rows * cols // gate.numel() + 2) * tn.abs().reshape(shape).sum(1)
        dgate = tuple(t.reshape(gate.shape) for t in dgate)
    v = total * g
    tol_v = tol * g.abs() + 2 * U * v.abs()
    dx = v, tol_v
    if post is not None:
        dx, dpost, dpost_bias = _norm_bwd(v, tol_v, xd, st[:, 0], st[:, 1],
                                          post.double() + offset, layer)
    out = [dx, (total, tol), dgate, dpost, None if post_bias is None else dpost_bias, dpre,
           None if pre_bias is None else dpre_bias]
    return [None if t is None else (t[0], rounded(t[0], t[1], x.dtype)) for t in out]


def _logits(hidden, weight, scale):
    """s, |s|'s sum of absolute products, and s's bound.  A matrix instruction
    may cut its sums instead of rounding them: a whole step, 2 U, for each of
    `width` additions; three products of parts that are left out of fp32
    operands are below 2^-24 each, and each part may add its own pass's roundings."""
    h, w = hidden.double(), weight.double()
    s = h @ w.t() * scale
    size = h.abs() @ w.abs().t() * scale
    return s, 2 * U * (h.shape[1] + 16) * size + 2 * U * s.abs() + 2.0 ** -140


def linear_cross_entropy(hidden, weight, tokens, scale=1.0, ignore_index=IGNORE):
    """(loss, lse) and their bounds."""
    s, tol_s = _logits(hidden, weight, f32(scale))
    vocab = s.shape[1]
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    m = s.amax(-1, keepdim=True)
    # Of e^(s - m): its difference, and 4 for the exponential and a rescaling;
    # the sum of a tile's 256 terms and of the tiles.
    adds = vocab / 256 + 40 + 8 * 4
    tol_lse = (p * (tol_s + U * (2 * (s - m).abs() + 6))).sum(-1) + U * (adds + 2 * lse.abs()
                                                                        + 2 * m[:, 0].abs() + 8)
    toks = tokens.long()
    skip, known = toks == ignore_index, (toks >= 0) & (toks < vocab)
    at = torch.where(known, toks, 0)[:, None]
    loss = lse - s.gather(1, at)[:, 0]
    tol_loss = tol_lse + tol_s.gather(1, at)[:, 0] + U * (loss.abs() + lse.abs())
    loss = torch.where(known, loss, torch.full_like(loss, NAN))
    return [(torch.where(skip, 0.0, v).cpu(), t.cpu()) for v, t in ((loss, tol_loss),
                                                                   (lse, tol_lse))]


def linear_cross_entropy_bwd(grad, hidden, weight, tokens, lse, scale=1.0, ignore_index=IGNORE,
                             grad_lse=None):
    """(dhidden, dweight) and their bounds, of the same lse."""
    scale = f32(scale)
    toks = tokens.long()
    keep = toks != ignore_index
    hidden_k = torch.where(keep[:, None], hidden.double(), 0.0)  # whatever they hold
    s, tol_s = _logits(hidden_k, weight, scale)
    vocab = s.shape[1]
    g = grad.double()[:, None]
    both = g if grad_lse is None else g + grad_lse.double()[:, None]
    lp = s - lse.double()[:, None]
    p = torch.exp(lp)
    hot = (torch.arange(vocab, device=toks.device)[None] == toks[:, None]).double()
    d = (both * p - hot * g) * scale
    size = both.abs() * p
    tol_d = scale * (size * (torch.expm1(tol_s + U * (2 * lp.abs() + 12))) + 3 * U * (
        size + hot * g.abs())) + U * d.abs() + 2.0 ** -126 * (1 + both.abs())
    if hidden.dtype == BF16:
        tol_d = tol_d + HALF[BF16] * (d.abs() + tol_d) + 2.0 ** -133
    k = keep[:, None].double()
    d, tol_d = d * k, tol_d * k
    w, wa, ha = weight.double(), weight.double().abs(), hidden_k.abs()
    adds = 2 * U * (vocab + 64)
    dh, tol_dh = d @ w, tol_d @ wa + adds * (d.abs() @ wa)
    adds = 2 * U * (len(toks) + 64)
    dw, tol_dw = d.t() @ hidden_k, tol_d.t() @ ha + adds * (d.abs().t() @ ha)
    unknown = keep & ((toks < 0) | (toks >= vocab))
    dh = torch.where(unknown[:, None], torch.full_like(dh, NAN), dh)
    if bool(unknown.any()):
        dw = torch.full_like(dw, NAN)
    return [(v.cpu(), rounded(v, t, hidden.dtype).cpu()) for v, t in ((dh, tol_dh), (dw, tol_dw))]
