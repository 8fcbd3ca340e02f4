"""The norms around a block and the output layer's cross entropy on the GPU
against the 64-bit reference, at the sizes, types and options where they could
go wrong; refusals; streams, graphs and a run of all of them together."""
import pytest
import torch

import block_ops_reference as ref
import fp32_parts_reference as parts

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NAN, INF, IGNORE = ref.NAN, ref.INF, ref.IGNORE
DTYPES = [BF16, F32]


@pytest.fixture(scope="module")
def ho():
    import hip_oracles
    hip_oracles.load_library()
    return hip_oracles


def shifted(t, shift):
    """t at `shift` values past an allocation's start, with NaN around it."""
    if t is None or not shift:
        return t
    buf = torch.full((t.numel() + 2 * shift,), NAN, dtype=t.dtype, device=t.device)
    view = buf[shift:shift + t.numel()].view(t.shape)
    view.copy_(t)
    return view


# ---------------------------------------------------------------------------
# Norms
# ---------------------------------------------------------------------------

def norm_operands(dev, rows, cols, dtype, *, norm, post=True, pre=True, gates=0, seed=0, shift=0,
                  scale=0.5, offset=1.0, bias=None):
    g = torch.Generator(device=dev).manual_seed(seed)

    def make(*shape, mean=0.0, std=1.0):
        t = (mean + std * torch.randn(*shape, generator=g, device=dev)).to(dtype)
        return shifted(t, shift)

    rowsof = dict(x=make(rows, cols, mean=0.3), residual=make(rows, cols, mean=-1.0, std=3.0))
    kw = dict(norm=norm, scale=scale, offset=offset)
    for name, there in (("post", post), ("pre", pre)):
        if there:
            kw[name] = make(cols, std=0.3)
            if norm == "layer" if bias is None else bias:
                kw[name + "_bias"] = make(cols, std=0.3)
    if gates:
        kw["gate"] = make(gates, cols, std=0.7)
        if gates == 1:
            kw["gate"] = kw["gate"][0]
    grads = dict(grad_h=make(rows, cols), grad_y=make(rows, cols) if pre else None)
    return rowsof, kw, grads


def check_norms(ho, rowsof, kw, grads, what, eps=1e-6):
    h, y, stats = ho.block_norms(**rowsof, **kw, eps=eps)
    want_h, tol_h, stats0, tol0 = ref.stream(**rowsof, **kw, eps=eps)
    c = lambda t: t.cpu()  # noqa: E731
    ref.close(h, c(want_h), c(tol_h), f"{what} h")
    ref.close(stats[:, :2], c(stats0), c(tol0), f"{what} statistics of x")
    if "pre" in kw:
        want_y, tol_y, stats1, tol1 = ref.after(h, **kw, eps=eps)
        ref.close(y, c(want_y), c(tol_y), f"{what} y")
        ref.close(stats[:, 2:], c(stats1), c(tol1), f"{what} statistics of h")
    else:
        assert y is None
    args = (grads["grad_h"], grads["grad_y"], rowsof["x"], h if "pre" in kw else None, stats)
    got = ho.block_norms_bwd(*args, **kw)
    want = ref.block_norms_bwd(*args, **kw)
    names = ("dx", "dresidual", "dgate", "dpost", "dpost_bias", "dpre", "dpre_bias")
    for name, u, v in zip(names, got, want):
        if v is None:
            assert u is None, name
            continue
        assert u.dtype == rowsof["x"].dtype
        ref.close(u, c(v[0]), c(v[1]), f"{what} {name}")
    return (h, y, stats), got


SIZES = [(1, 8), (1, 9), (3, 15), (65, 16), (7, 64), (300, 100), (33, 504), (40, 511), (1000, 512),
         (40, 513), (7, 520), (2, 1001), (515, 1024), (17, 1025), (20, 2880), (9, 4096), (5, 5000),
         (3, 8192), (3, 8193), (2, 16383), (6, 16384)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_norms_sizes(rows, cols, norm, dtype, rocm_device, ho):
    for k, (post, pre, gates, shift) in enumerate(
            ((True, True, 0, 0), (True, False, 1, 1), (False, True, rows, 3), (True, True, 1, 0))):
        case = norm_operands(rocm_device, rows, cols, dtype, norm=norm, post=post, pre=pre,
                             gates=gates, shift=shift, seed=k)
        if k == 3 and pre:
            case[2]["grad_h"] = None
        check_norms(ho, *case, f"[{rows}, {cols}] {dtype} {norm} {k}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [64, 700, 2880])
@pytest.mark.parametrize("rows,gates", [(6, 2), (6, 3), (4096, 2), (4096, 3), (4096, 7), (4096, 16),
                                        (4096, 64), (4096, 512), (4096, 1024), (4096, 4096),
                                        (2050, 41), (8190, 30)])
def test_gates_of_samples(rows, gates, cols, dtype, rocm_device, ho):
    """Rows of a gate within a workgroup, over several, and both at once."""
    rows = rows // gates * gates
    for norm, post in (("layer", True), ("rms", False)):
        case = norm_operands(rocm_device, rows, cols, dtype, norm=norm, post=post, gates=gates,
                             scale=1.0, offset=0.0)
        check_norms(ho, *case, f"[{rows}, {cols}] {gates} gates {dtype} {norm}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,gates,cols", [(600, 7, 9001), (600, 600, 12288), (1024, 16, 16384),
                                             (1024, 512, 8200)])
def test_gates_of_wide_samples(rows, gates, cols, dtype, rocm_device, ho):
    test_gates_of_samples(rows, gates, cols, dtype, rocm_device, ho)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("rows,cols", [(30011, 64), (9001, 1001), (8192, 2048), (700, 8192),
                                       (777, 9001), (520, 16384)])
def test_norms_of_many_rows(rows, cols, norm, dtype, rocm_device, ho):
    """The same bits again, biases left out, and rows that are the same in
    another batch."""
    for gates in (0, 1):
        case = norm_operands(rocm_device, rows, cols, dtype, norm=norm, gates=gates,
                             bias=gates == 0 and norm == "layer")
        first, grads = check_norms(ho, *case, f"[{rows}, {cols}] {dtype} {norm} {gates}")
        again = ho.block_norms(**case[0], **case[1])
        some = slice(rows // 3, rows // 2)
        part = ho.block_norms(*(v[some].contiguous() for v in case[0].values()), **case[1])
        for a, b, p in zip(first, again, part):
            assert torch.equal(a, b) and torch.equal(a[some], p)
        args = (case[2]["grad_h"], case[2]["grad_y"], case[0]["x"], first[0], first[2])
        for a, b in zip(grads, ho.block_norms_bwd(*args, **case[1])):
            assert (a is None and b is None) or torch.equal(a, b)
        part = ho.block_norms_bwd(*(v[some].contiguous() for v in args), **case[1])
        assert torch.equal(part[0], grads[0][some]) and torch.equal(part[1], grads[1][some])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [40, 1100])
def test_norms_of_special_rows(cols, dtype, rocm_device, ho):
    """Zero and constant rows, NaN, infinities: in their own rows only."""
    rows = 12
    for norm in ("rms", "layer"):
        rowsof, kw, grads = norm_operands(rocm_device, rows, cols, dtype, norm=norm, gates=rows)
        x, r = rowsof["x"], rowsof["residual"]
        clean = ho.block_norms(x, r, **kw)
        x[1] = 0.0
        x[2] = 1.5
        r[3] = 0.0
        x[3] = 0.0
        x[4, cols // 2] = NAN
        r[5, 0] = NAN
        x[6, cols - 1] = INF
        r[7, cols // 3] = -INF
        h, y, stats = ho.block_norms(x, r, **kw)
        for k in (0, 8, 9, 10, 11):
            assert torch.equal(h[k], clean[0][k]) and torch.equal(y[k], clean[1][k])
        assert torch.isfinite(y[[1, 2, 3]]).all()
        assert h[4].isnan().all() and y[4].isnan().all()
        assert h[5].isnan().sum() == 1 and y[5].isnan().all()
        assert y[6].isnan().all() and y[7].isnan().any()
        fine = [0, 1, 2, 3, 8, 9, 10, 11]
        part = {k: v[fine].contiguous() for k, v in rowsof.items()}
        kwp = {**kw, "gate": kw["gate"][fine].contiguous()}
        check_norms(ho, part, kwp, {k: v[fine].contiguous() for k, v in grads.items()},
                    f"{cols} {dtype} {norm}")
        got = ho.block_norms_bwd(grads["grad_h"], grads["grad_y"], x, h, stats, **kw)
        want = ho.block_norms_bwd(*(v[fine].contiguous() for v in (
            grads["grad_h"], grads["grad_y"], x, h, stats)), **kwp)
        for k in range(3):  # rows of their own
            assert torch.equal(got[k][fine], want[k])
        assert got[0][4].isnan().all() and got[3].isnan().any()


def test_norms_beside_those_of_the_library(rocm_device, ho):
    """Without a norm before the sum, a gate or a scale: residual_layernorm and
    rmsnorm_ex."""
    g = torch.Generator(device=rocm_device).manual_seed(1)
    x, r = (torch.randn(70, 1024, generator=g, device=rocm_device).to(BF16) for _ in range(2))
    w, b = (torch.randn(1024, generator=g, device=rocm_device).to(BF16) for _ in range(2))
    h, y, _ = ho.block_norms(x, r, pre=w, pre_bias=b, norm="layer", eps=1e-5)
    h2, y2, _, _ = ho.residual_layernorm(x, r, w, b, 1e-5)
    assert torch.equal(h, h2)
    torch.testing.assert_close(y.float(), y2.float(), rtol=2.0 ** -7, atol=1e-5)
    h, y, _ = ho.block_norms(x, r, pre=w, eps=1e-5)
    h2, y2 = ho.rmsnorm_ex(x, w, 1e-5, residual=r, want_h=True)
    assert torch.equal(h, h2)
    torch.testing.assert_close(y.float(), y2.float(), rtol=2.0 ** -7, atol=1e-6)


def test_norms_without_rows(rocm_device, ho):
    x = torch.zeros(0, 64, device=rocm_device)
    w = torch.ones(64, device=rocm_device)
    h, y, stats = ho.block_norms(x, x, post=w, pre=w, gate=w)
    assert h.shape == y.shape == (0, 64) and stats.shape == (0, 4)
    out = ho.block_norms_bwd(x, x, x, h, stats, post=w, pre=w, gate=w)
    assert out[0].shape == out[1].shape == (0, 64)
    assert all(not t.any() for t in (out[2], out[3], out[5]))


def test_norms_refuse(rocm_device, ho):
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device=rocm_device)  # noqa: E731
    x, w, st = z(4, 16), z(16), z(4, 4, t=F32)
    for call, msg in [
            (lambda: ho.block_norms(x, x), "norm is needed"),
            (lambda: ho.block_norms(x.half(), x.half(), pre=w.half()), "bf16 or fp32"),
            (lambda: ho.block_norms(x, x.float(), pre=w), "one type"),
            (lambda: ho.block_norms(x, z(4, 8), pre=w), "contiguous"),
            (lambda: ho.block_norms(z(16, 4).t(), x, pre=w), "contiguous"),
            (lambda: ho.block_norms(x, x, pre=w.float()), "rows' type"),
            (lambda: ho.block_norms(x, x, pre=z(32)[::2]), "contiguous"),
            (lambda: ho.block_norms(x, x, pre=w, gate=z(3, 16)), "divide"),
            (lambda: ho.block_norms(x, x, pre=w, gate=z(4, 8)), "gate"),
            (lambda: ho.block_norms(x, x, pre=w, gate=z(())), "gate"),
            (lambda: ho.block_norms(x, x, pre=w, gate=z(2, 2, 16)), "gate"),
            (lambda: ho.block_norms(x, x, pre=w, norm="batch"), "norm must be"),
            (lambda: ho.block_norms_bwd(x, None, x, x, st, pre=w), "go together"),
            (lambda: ho.block_norms_bwd(x, x, x, None, st, pre=w), "go together"),
            (lambda: ho.block_norms_bwd(x, x, x, x, st, post=w), "go together"),
            (lambda: ho.block_norms_bwd(None, None, x, None, st, post=w), "no gradient"),
            (lambda: ho.block_norms_bwd(x, x, x, x, z(4, 2, t=F32), pre=w), "stats"),
            (lambda: ho.block_norms_bwd(x, x, x, x, st.double(), pre=w), "stats")]:
        with pytest.raises((ValueError, RuntimeError), match=msg):
            call()
    for kw, msg in [(dict(pre=w, pre_bias=w), "LayerNorm"), (dict(pre=w, scale=INF), "finite"),
                    (dict(pre=w, eps=-1.0), "eps")]:
        with pytest.raises(RuntimeError, match=msg):
            ho.block_norms(x, x, **kw)
    with pytest.raises(RuntimeError, match="cols"):
        ho.block_norms(z(4, 7), z(4, 7), pre=z(7))
    with pytest.raises(RuntimeError, match="cols"):
        ho.block_norms(z(1, 16385), z(1, 16385), pre=z(16385))


# ---------------------------------------------------------------------------
# Cross entropy
# ---------------------------------------------------------------------------

def layer_operands(dev, rows, width, vocab, dtype, *, seed=0, pads=(0, 0), shift=0, std=2.5):
    g = torch.Generator(device=dev).manual_seed(seed)

    def make(n, pad, scale):
        t = torch.full((n * (width + pad) + shift,), NAN, dtype=dtype, device=dev)
        t = t[shift:].view(n, width + pad)[:, :width]
        t.copy_((torch.randn(n, width, generator=g, device=dev) * scale).to(dtype))
        return t

    hidden, weight = make(rows, pads[0], 1.0), make(vocab, pads[1], std / width ** 0.5)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    grads = torch.randn(2, rows, generator=g, device=dev)
    return hidden, weight, tokens, grads


def check_loss(ho, hidden, weight, tokens, grads, what, scale=1.0, wide=True):
    t = tokens if wide else tokens.to(torch.int32)
    got = ho.linear_cross_entropy(hidden, weight, t, scale=scale)
    want = ref.linear_cross_entropy(hidden, weight, tokens, scale)
    for name, u, (v, tol) in zip(("loss", "lse"), got, want):
        ref.close(u, v, tol, f"{what} {name}")
    lse = got[1]
    for gl in (None, grads[1]):
        out = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, t, lse, scale=scale,
                                          grad_lse=gl)
        wanted = ref.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse, scale,
                                              grad_lse=gl)
        for name, u, (v, tol) in zip(("dhidden", "dweight"), out, wanted):
            assert u.dtype == hidden.dtype and u.is_contiguous()
            ref.close(u, v, tol, f"{what} {name}")
    return got, out


LAYERS = [(1, 1, 1), (1, 8, 2), (2, 3, 5), (1, 64, 255), (3, 72, 256), (16, 64, 257), (17, 128, 1000),
          (5, 1001, 3001), (32, 1032, 777), (33, 200, 700), (48, 2056, 129), (64, 96, 2000),
          (64, 1024, 1025), (65, 512, 513), (100, 65, 4097), (128, 264, 640), (200, 1000, 260),
          (129, 64, 1023), (256, 128, 512), (257, 64, 513), (300, 320, 1500), (515, 777, 1030),
          (1000, 40, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", LAYERS)
def test_cross_entropy_sizes(rows, width, vocab, dtype, rocm_device, ho):
    for k, (pads, shift, scale) in enumerate((((0, 0), 0, 1.0), ((8, 16), 0, 0.7),
                                              ((3, 5), 1, 1.25))):
        case = layer_operands(rocm_device, rows, width, vocab, dtype, pads=pads, shift=shift,
                              seed=k)
        check_loss(ho, *case, f"[{rows}, {width}, {vocab}] {dtype} {k}", scale, wide=k != 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 20, 70, 300, 1030, 2500])
@pytest.mark.parametrize("kind", ["some", "all", "but one", "first", "last", "unknown"])
def test_cross_entropy_of_rows_left_out(kind, rows, dtype, rocm_device, ho):
    """Rows of ignore_index count nowhere, whatever they hold."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, 72, 600, dtype)
    out = torch.zeros(rows, dtype=torch.bool, device=rocm_device)
    if kind == "some":
        out[::3] = True
    elif kind == "all":
        out[:] = True
    elif kind == "but one":
        out[:] = True
        out[rows // 2] = False
    elif kind == "first":
        out[:rows // 2] = True
    elif kind == "last":
        out[rows // 2:] = True
    tokens[out] = IGNORE
    hidden[out] = NAN
    if rows > 2:
        hidden[out.nonzero()[:1, 0]] = INF
    if kind == "unknown":
        tokens[0], tokens[rows // 2] = 600, -1
    check_loss(ho, hidden, weight, tokens, grads, f"{kind} {rows} {dtype}")
    if kind in ("some", "first"):
        other = ho.linear_cross_entropy(hidden, weight, torch.where(out, 5, tokens), ignore_index=5)
        kept = ~out & (tokens != 5)
        assert torch.equal(other[0][kept], ho.linear_cross_entropy(hidden, weight, tokens)[0][kept])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [(3, 4096, 20011), (1, 2048, 32000), (700, 1024, 9001),
                                              (2100, 256, 33000), (40, 264, 100003),
                                              (20, 512, 17001), (64, 192, 24000)])
def test_cross_entropy_of_larger_layers(rows, width, vocab, dtype, rocm_device, ho):
    case = layer_operands(rocm_device, rows, width, vocab, dtype, std=5.0)
    what = f"[{rows}, {width}, {vocab}] {dtype}"
    got, out = check_loss(ho, *case, what, 0.7)
    hidden, weight, tokens, grads = case
    again = ho.linear_cross_entropy(hidden, weight, tokens, scale=0.7)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), what
    again = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, got[1], scale=0.7,
                                        grad_lse=grads[1])
    assert all(torch.equal(a, b) for a, b in zip(out, again)), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [(3, 8, 5 << 20), (3, 9, 7 << 20), (400, 64, 1 << 21)])
def test_gradients_over_pieces_of_the_vocabulary(rows, width, vocab, dtype, rocm_device, ho):
    """More of the vocabulary than one piece of the workspace holds: 1.5 GB of d,
    of few rows and of more."""
    vocab += 77
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, vocab, dtype)
    loss, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    logits = hidden.double() @ weight.double().t()
    want = torch.logsumexp(logits, -1)
    assert float((lse - want).abs().max()) < 1e-5  # lse below 32: 4 steps of 2^-19
    dh, dw = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse)
    # The bound of the sum over the vocabulary is wide; in the mean its roundings
    # cancel.  A wrong piece shows in the norm of what it holds.
    d = torch.exp(logits - lse[:, None].double()) * grads[0][:, None].double()
    del logits
    d[torch.arange(rows), tokens] -= grads[0].double()
    least = 2.0 ** -7 if dtype == BF16 else 2.0 ** -18
    for got, whole in ((dh, d @ weight.double()), (dw, d.t() @ hidden.double())):
        assert float((got.double() - whole).norm() / whole.norm()) < least
    part = dw.double().view(-1)[:width * (vocab // 64 * 64)].view(64, -1).norm(dim=-1)
    whole = (d.t() @ hidden.double())[:vocab // 64 * 64].reshape(64, -1).norm(dim=-1)
    assert float(((part - whole) / whole).abs().max()) < least


def test_losses_over_pieces_of_the_vocabulary(rocm_device, ho):
    """More fp32 weights than the 1 GB of copies that one piece of the workspace is."""
    hidden, weight, tokens, _ = layer_operands(rocm_device, 70, 1024, 180001, F32)
    got = ho.linear_cross_entropy(hidden, weight, tokens, scale=0.7)
    for name, u, (v, tol) in zip(("loss", "lse"), got, ref.linear_cross_entropy(
            hidden, weight, tokens, 0.7)):
        ref.close(u, v, tol, name)


@pytest.mark.parametrize("rows,width", [(1, 64), (1, 65), (3, 200), (20, 72), (64, 131)])
def test_gradients_of_few_rows_are_rounded_once(rows, width, rocm_device, ho):
    """Up to 64 rows d has two bf16 parts, so that bf16 gradients are off by their
    own rounding alone: half a step, and 2^-15 of the sums of absolute products
    for the parts' and the sums' own."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, 1500, BF16)
    _, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    got = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse)
    h, w = hidden.double(), weight.double()
    d = torch.exp(h @ w.t() - lse[:, None].double()) * grads[0][:, None].double()
    d[torch.arange(rows), tokens] -= grads[0].double()
    for u, v, size in ((got[0], d @ w, d.abs() @ w.abs()),
                       (got[1], d.t() @ h, d.abs().t() @ h.abs())):
        ref.close(u, v.cpu(), (v.abs() * 2.0 ** -8 + size * 2.0 ** -15).cpu(), f"{rows} {width}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [6, 300])
def test_cross_entropy_of_special_values(rows, dtype, rocm_device, ho):
    """Rows with NaN and infinities are alone with them; logits far from zero and
    far apart; weights of rows that are NaN."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, 64, 700, dtype)
    clean = ho.linear_cross_entropy(hidden, weight, tokens)
    bad = hidden.clone()
    bad[1, 5] = NAN
    bad[2] = INF
    got = ho.linear_cross_entropy(bad, weight, tokens)
    keep = [k for k in range(rows) if k not in (1, 2)]
    for a, b in zip(clean, got):
        assert torch.equal(a[keep], b[keep])
        assert b[1].isnan() and not torch.isfinite(b[2])
    dh, _ = ho.linear_cross_entropy_bwd(grads[0], bad, weight, tokens, got[1])
    want, _ = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, clean[1])
    assert torch.equal(dh[keep], want[keep]) and dh[1].isnan().all()
    check_loss(ho, hidden * 40, weight, tokens, grads, f"far apart {rows} {dtype}")
    one = torch.zeros_like(hidden)
    one[:, 0] = 1.0
    up = weight.clone()
    up[:, 0] += 3e4
    check_loss(ho, one, up, tokens, grads, f"far from zero {rows} {dtype}")
    check_loss(ho, torch.zeros_like(hidden), weight, tokens, grads, f"equal {rows} {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_losses_of_logits_in_memory(dtype, rocm_device, ho):
    """token_logprobs of the logits, where they are exact: small whole numbers."""
    g = torch.Generator(device=rocm_device).manual_seed(4)
    hidden = torch.randint(-2, 3, (90, 24), generator=g, device=rocm_device).to(dtype)
    weight = torch.randint(-2, 3, (1500, 24), generator=g, device=rocm_device).to(dtype)
    t = torch.randint(0, 1500, (90,), generator=g, device=rocm_device)
    t[::9] = IGNORE
    logits = (hidden.float() @ weight.float().t()).to(dtype)
    loss, lse = ho.linear_cross_entropy(hidden, weight, t, scale=0.5)
    lp, lse2 = ho.token_logprobs(logits, t, scale=0.5)
    assert float((loss + lp).abs().max()) < 2e-5 and float((lse - lse2).abs().max()) < 2e-5


def test_cross_entropy_without_rows(rocm_device, ho):
    h = torch.zeros(0, 16, device=rocm_device)
    w, t, f = torch.ones(20, 16, device=rocm_device), torch.zeros(
        0, dtype=torch.int64, device=rocm_device), torch.zeros(0, device=rocm_device)
    loss, lse = ho.linear_cross_entropy(h, w, t)
    assert loss.shape == lse.shape == (0,)
    dh, dw = ho.linear_cross_entropy_bwd(f, h, w, t, f)
    assert dh.shape == (0, 16) and dw.shape == (20, 16) and not dw.any()


def test_cross_entropy_refuses(rocm_device, ho):
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device=rocm_device)  # noqa: E731
    h, w, t, f = z(4, 16), z(9, 16), z(4, t=torch.int64), z(4, t=F32)
    for call, msg in [
            (dict(hidden=h.half()), "bf16 or fp32"), (dict(weight=w.float()), "hidden's type"),
            (dict(weight=z(9, 8)), "hidden's type"), (dict(tokens=f), "tokens"),
            (dict(tokens=t[:3]), "tokens"), (dict(scale=0.0), "scale"),
            (dict(scale=NAN), "scale"), (dict(weight=z(0, 16)), "empty"),
            (dict(hidden=z(16, 4).t()), "inner"), (dict(weight=z(16, 9).t()), "inner"),
            (dict(hidden=z(1, 16).expand(4, 16)), "overlap"),
            (dict(weight=z(1, 16).expand(9, 16)), "overlap"), (dict(lse=z(4)), "fp32"),
            (dict(grad=z(3, t=F32)), "fp32"), (dict(grad_lse=z(8, t=F32)[::2]), "fp32")]:
        args = {"hidden": h, "weight": w, "tokens": t, **call}
        with pytest.raises(ValueError, match=msg):
            ho.linear_cross_entropy_bwd(**{"grad": f, "lse": f, **args})
        if not {"lse", "grad", "grad_lse"} & set(call):
            with pytest.raises(ValueError, match=msg):
                ho.linear_cross_entropy(**args)


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------

class Model:
    """Two residual blocks (a product each) between an embedding and the loss,
    weights tied, and their gradients, all through the library."""

    def __init__(self, ho, dev, rows, width, vocab, dtype, seed=0):
        g = torch.Generator(device=dev).manual_seed(seed)
        make = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=dev) * std).to(dtype)  # noqa: E731
        self.ho, self.rows, self.vocab, self.dtype = ho, rows, vocab, dtype
        self.table = make(vocab, width)
        self.blocks = [make(width, width, std=width ** -0.5) for _ in range(2)]
        self.norms = [dict(post=make(width, std=0.1), pre=make(width, std=0.1), gate=make(
            4, width, std=0.5)) for _ in range(2)]
        self.ids = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        self.next = torch.randint(0, vocab, (rows,), generator=g, device=dev)
        self.next[::5] = IGNORE
        self.grad = torch.full((rows,), 1.0 / rows, device=dev)

    def step(self):
        ho, kw = self.ho, dict(offset=1.0, scale=0.7)
        h = ho.embedding(self.table, self.ids)
        y, kept = h, []
        for w, n in zip(self.blocks, self.norms):
            x = y @ w
            h, out, stats = ho.block_norms(x, h, **n, **kw)
            kept.append((y, x, h, stats))
            y = out
        width = y.shape[1]
        loss, lse = ho.linear_cross_entropy(y, self.table, self.next, scale=width ** -0.5)
        dy, dtable = ho.linear_cross_entropy_bwd(self.grad, y, self.table, self.next, lse,
                                                 scale=width ** -0.5)
        dh, out = None, [loss]
        for (y, x, h, stats), w, n in zip(kept[::-1], self.blocks[::-1], self.norms[::-1]):
            dx, dh, *dn = ho.block_norms_bwd(dh, dy, x, h, stats, **n, **kw)
            out += [y.t() @ dx, *(t for t in dn if t is not None)]
            dy = dx @ w.t()
        demb = (dh.float() + dy.float()).to(self.dtype)
        out.append(ho.embedding_bwd(demb, self.ids, self.vocab, into=dtable))
        return out

    def exact(self):
        """The same by automatic differentiation in 64 bits."""
        leaf = lambda t: t.double().requires_grad_()  # noqa: E731
        table, blocks = leaf(self.table), [leaf(w) for w in self.blocks]
        norms = [{k: leaf(v) for k, v in n.items()} for n in self.norms]
        h = table[self.ids]
        y = h
        width = h.shape[1]
        for w, n in zip(blocks, norms):
            x = y @ w
            x = torch.nn.functional.rms_norm(x, (width,), 1.0 + n["post"], 1e-6)
            h = h + 0.7 * x * n["gate"].repeat_interleave(self.rows // 4, 0)
            y = torch.nn.functional.rms_norm(h, (width,), 1.0 + n["pre"], 1e-6)
        loss = torch.nn.functional.cross_entropy(y @ table.t() * width ** -0.5, self.next,
                                                 ignore_index=IGNORE, reduction="none")
        (loss * self.grad.double()).sum().backward()
        out = [loss.detach()]
        for w, n in zip(blocks[::-1], norms[::-1]):
            out += [w.grad, n["gate"].grad, n["post"].grad, n["pre"].grad]
        return out + [table.grad]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [(40, 64, 300), (260, 520, 2003)])
def test_a_run_of_them_together(rows, width, vocab, dtype, rocm_device, ho):
    """bf16 values between the calls are off by 2^-8 each, of a chain of some 16
    roundings; fp32 by 2^-24 of sums of `width` and more terms."""
    m = Model(ho, rocm_device, rows, width, vocab, dtype)
    least = 16 * 2.0 ** -8 if dtype == BF16 else 2.0 ** -24 * 16 * width
    for k, (u, v) in enumerate(zip(m.step(), m.exact())):
        assert u.shape == v.shape
        assert float((u.double() - v).norm() / v.norm()) < least, k


@pytest.mark.parametrize("rows", [40, 1100])
def test_the_run_in_a_graph(rows, rocm_device, ho):
    """Captured once and replayed on new tokens, another number of them left
    out, with eager work between."""
    m = Model(ho, rocm_device, rows, 128, 2003, BF16)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        m.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = m.step()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        m.ids.copy_(torch.randint(0, m.vocab, m.ids.shape, generator=g))
        m.next.copy_(torch.randint(0, m.vocab, m.next.shape, generator=g))
        m.next[:seed * rows // 3] = IGNORE
        eager = [v.clone() for v in m.step()]
        graph.replay()
        torch.cuda.synchronize()
        for k, (u, v) in enumerate(zip(captured, eager)):
            assert torch.equal(u, v), f"replay {seed}, output {k}"


def test_two_streams_at_once(rocm_device, ho):
    models = [Model(ho, rocm_device, 600, 256, 5000, BF16, seed=k) for k in range(2)]
    want = [[v.clone() for v in m.step()] for m in models]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in models]
    for _ in range(3):
        got = []
        for m, s in zip(models, streams):
            with torch.cuda.stream(s):
                got.append(m.step())
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def gradients_in_64_bits(grad, hidden, weight, tokens, lse, scale=1.0):
    """[(dhidden or dweight, the sums of its absolute products)] of one lse."""
    h, w = hidden.double(), weight.double()
    keep = tokens != IGNORE
    d = torch.exp(h @ w.t() * scale - lse[:, None].double()) * grad[:, None].double()
    d[keep.nonzero()[:, 0], tokens[keep]] -= grad[keep].double()
    d *= scale * keep[:, None]
    return [(d @ w, d.abs() @ w.abs()), (d.t() @ h, d.abs().t() @ h.abs())]


@pytest.mark.parametrize("rows,width,vocab", [
    (64, 264, 1500), (65, 264, 1500), (65, 65, 1501), (200, 1000, 260), (700, 768, 9001),
    (1030, 72, 4000), (2500, 520, 8000), (400, 64, (1 << 20) + 77)])
def test_gradients_of_two_parts_are_rounded_once(rows, width, vocab, rocm_device, ho):
    """With two_parts bf16 gradients are off by their own rounding alone: half a
    step of each, and in the 2-norm what rounding the 64-bit gradients is off by.
    d's two parts leave 2^-16 of it at most, so 2^-15 of the sums of absolute
    products with the sums' own roundings; in the norm, where these have either
    sign, 2^-14 of the gradient, a twentieth of the 2^-9.2 that the rounding is.
    One part is off by as much as the rounding, 1.4 times as much in all.  (The
    last size is two pieces of the vocabulary.)"""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, vocab, BF16)
    tokens[::9] = IGNORE
    _, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    args = (grads[0], hidden, weight, tokens, lse)
    want = gradients_in_64_bits(*args)
    got = ho.linear_cross_entropy_bwd(*args, two_parts=True)
    again = ho.linear_cross_entropy_bwd(*args, two_parts=True)
    one = ho.linear_cross_entropy_bwd(*args)
    for name, u, a, o, (v, size) in zip(("dhidden", "dweight"), got, again, one, want):
        what = f"[{rows}, {width}, {vocab}] {name}"
        assert torch.equal(u, a), what
        own = float((v.to(BF16).double() - v).norm())
        off = float((u.double() - v).norm())
        assert off <= 1.05 * own, f"{what}: {off / own:.3f} of the rounding"
        if rows <= 64:
            assert torch.equal(u, o), what
        over = (u.double() - v).abs() - v.abs() * 2.0 ** -8 - size * 2.0 ** -15
        assert float(over.max()) <= 2.0 ** -133, what


def test_two_parts_of_fp32_are_three(rocm_device, ho):
    hidden, weight, tokens, grads = layer_operands(rocm_device, 100, 72, 900, F32)
    _, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    got = [ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse, two_parts=k)
           for k in (False, True)]
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("elem,dtype", [(2, BF16), (4, F32)])
@pytest.mark.parametrize("width,vocab", [(1, 1), (7, 3), (65, 1001), (264, 2000)])
def test_the_gradient_of_no_rows_is_zero(width, vocab, elem, dtype, rocm_device, ho):
    """As of rows that are all left out, and no value beside dweight is written."""
    lib = ho.load_library()
    for bwd in (lib.hipo_linear_cross_entropy_bwd, lib.hipo_linear_cross_entropy_bwd_two_parts):
        for shift in (64, 65):
            buf = torch.full((width * vocab + 2 * shift,), NAN, dtype=dtype, device=rocm_device)
            rc = bwd(None, None, None, elem, None, 8, None, None, None,
                     buf.data_ptr() + shift * elem, 0, width, vocab, width, width, 1.0, IGNORE,
                     None, 0, torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            assert not buf[shift:-shift].any()
            assert buf[:shift].isnan().all() and buf[-shift:].isnan().all()


@pytest.mark.parametrize("bad", [1.0, [0.0], "x"])
def test_what_is_no_tensor_is_refused(bad, rocm_device, ho):
    z = lambda *s, t=BF16: torch.zeros(*s, dtype=t, device=rocm_device)  # noqa: E731
    x, w, st = z(4, 16), z(16), z(4, 4, t=F32)
    t, f = z(4, t=torch.int64), z(4, t=F32)
    layer = dict(norm="layer", post=w, pre=w)
    calls = [lambda kw=kw: ho.block_norms(**{"x": x, "residual": x, **layer, **kw})
             for kw in (dict(x=bad), dict(residual=bad), dict(post=bad), dict(post_bias=bad),
                        dict(pre=bad), dict(pre_bias=bad), dict(gate=bad))]
    given = dict(grad_h=x, grad_y=x, x=x, h=x, stats=st)
    calls += [lambda kw=kw: ho.block_norms_bwd(**{**given, **layer, **kw})
              for kw in [{k: bad} for k in (*given, "post", "post_bias", "pre", "pre_bias",
                                            "gate")]]
    loss = dict(hidden=x, weight=x, tokens=t)
    calls += [lambda kw=kw: ho.linear_cross_entropy(**{**loss, **kw})
              for kw in [{k: bad} for k in loss]]
    loss_bwd = dict(loss, grad=f, lse=f, grad_lse=f)
    calls += [lambda kw=kw: ho.linear_cross_entropy_bwd(**{**loss_bwd, **kw})
              for kw in [{k: bad} for k in loss_bwd]]
    for k, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {k}")


# ---------------------------------------------------------------------------
# Products of fp32 values: every part of every value counts
# ---------------------------------------------------------------------------

def assert_near(got, want, tol, what):
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0, (
        f"{what}: {float((over > 0).double().mean()):.2%} of the values are over the bound, "
        f"{float(((got.double() - want).abs() / tol.clamp(min=1e-300)).max()):.2f} times it")


@pytest.mark.parametrize("size", parts.SIZES)
def test_parts_of_fp32_logits(size, rocm_device, ho):
    """lse is the row's one logit; the gradient's e^(s - lse) shows its own s."""
    hidden, weight, tokens, (h, w) = parts.one_logit_a_row(*size, rocm_device)
    s = h.double() * w.double()
    _, got = ho.linear_cross_entropy(hidden, weight, tokens)
    assert_near(got, s, parts.TOL * s.abs(), f"{size} lse")
    lse = s.float()
    p = torch.exp(s - lse.double())
    zero, one = torch.zeros_like(lse), torch.ones_like(lse)
    dh, _ = ho.linear_cross_entropy_bwd(zero, hidden, weight, tokens, lse, grad_lse=one)
    want = p[:, None] * weight[tokens].double()
    # Of e^: s's own bound, half a step of s - lse, below 2^-4, and of its product,
    # and a step of the exponential: 2^-22 in all, 2^-20 with the product's.
    tol = want.abs() * torch.expm1(parts.TOL * s.abs() + 2.0 ** -20)[:, None]
    assert_near(dh, want, tol, f"{size} dhidden")


@pytest.mark.parametrize("size", parts.SIZES)
def test_parts_of_fp32_gradients(size, rocm_device, ho):
    grad, hidden, weight, tokens, lse = parts.one_value_of_d_a_row(*size, rocm_device)
    dh, dw = ho.linear_cross_entropy_bwd(grad, hidden, weight, tokens, lse)
    d = -grad.double()[:, None]
    want = d * weight[tokens].double()
    assert_near(dh, want, parts.TOL * want.abs(), f"{size} dhidden")
    want = d * hidden.double()
    assert_near(dw[tokens], want, parts.TOL * want.abs(), f"{size} dweight")
    rest = torch.ones(size[2], dtype=torch.bool, device=rocm_device)
    rest[tokens] = False
    assert not dw[rest].any(), f"{size}: dweight of other tokens"


# ---------------------------------------------------------------------------
# Nothing is written beside the outputs and the workspace
# ---------------------------------------------------------------------------

class Fenced:
    """Memory of exactly the size asked for, `past` bytes behind a 16-byte
    boundary, full of NaN, with a pattern before and behind it."""
    FENCE, BYTE = 1 << 16, 0xA5

    def __init__(self, dev, size, past=0):
        self.from_, self.size = self.FENCE + past, size
        self.all = torch.full((size + 2 * self.FENCE + past,), self.BYTE, dtype=torch.uint8,
                              device=dev)
        self.all[self.from_:self.from_ + size] = 0xFF
        assert self.all.data_ptr() % 16 == 0

    def ptr(self):
        return self.all.data_ptr() + self.from_

    def holds(self, want):
        """Whether it has want's bits, and the pattern is as it was."""
        inside = self.all[self.from_:self.from_ + self.size]
        return torch.equal(inside, want.contiguous().view(-1).view(torch.uint8))

    def intact(self):
        before, behind = self.all[:self.from_], self.all[self.from_ + self.size:]
        return bool((before == self.BYTE).all() and (behind == self.BYTE).all())


def fenced_call(ho, fn, what, outputs, before, after, need, dev, past):
    """fn(*before, *outputs, *after[, workspace, its size], stream) with the outputs
    (tensors of what they should be, or None) fenced."""
    outs = [None if t is None else Fenced(dev, t.numel() * t.element_size(), past) for t in outputs]
    ws = None if need is None else Fenced(dev, need)
    args = [*before, *(None if f is None else f.ptr() for f in outs), *after]
    if ws is not None:
        args += [ws.ptr(), need]
    rc = fn(*args, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, (what, ho.load_library().hipo_last_error())
    torch.cuda.synchronize()
    for k, (f, t) in enumerate(zip(outs, outputs)):
        if f is not None:
            assert f.intact(), f"{what}: written beside output {k}"
            assert f.holds(t), f"{what}: output {k}"
    assert ws is None or ws.intact(), f"{what}: written beside the workspace"


def address(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 9), (5, 15), (40, 511), (33, 520), (600, 700),
                                       (7, 1001), (17, 1025), (9, 2880), (3, 5000), (2, 8193),
                                       (2, 16383), (300, 16384)])
def test_norms_write_their_outputs_alone(rows, cols, dtype, rocm_device, ho):
    lib, elem = ho.load_library(), torch.finfo(dtype).bits // 8
    for k, (norm, post, pre, gates) in enumerate((
            ("layer", True, True, rows), ("rms", True, False, 1), ("layer", False, True, 0),
            ("rms", True, True, 1 if rows % 3 else rows // 3))):
        rowsof, kw, grads = norm_operands(rocm_device, rows, cols, dtype, norm=norm, post=post,
                                          pre=pre, gates=gates, seed=k)
        what, layer = f"[{rows}, {cols}] {dtype} {k}", int(norm == "layer")
        out = ho.block_norms(**rowsof, **kw)
        vectors = [address(kw.get(n)) for n in ("post", "post_bias", "pre", "pre_bias", "gate")]
        past = elem * k
        fenced_call(ho, lib.hipo_block_norms, what, out,
                    [address(rowsof["x"]), address(rowsof["residual"]), elem, *vectors],
                    [rows, cols, gates, kw["scale"], kw["offset"], 1e-6, layer], None,
                    rocm_device, past)
        h = out[0] if pre else None
        got = ho.block_norms_bwd(grads["grad_h"], grads["grad_y"], rowsof["x"], h, out[2], **kw)
        fenced_call(ho, lib.hipo_block_norms_bwd, f"{what} gradient", got,
                    [address(grads["grad_h"]), address(grads["grad_y"]), address(rowsof["x"]),
                     address(h), address(out[2]), elem, *vectors],
                    [rows, cols, gates, kw["scale"], kw["offset"], layer],
                    lib.hipo_block_norms_bwd_workspace_bytes(rows, cols), rocm_device, past)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [
    (1, 1, 1), (3, 72, 256), (5, 1001, 3001), (16, 64, 17000), (33, 200, 700), (64, 96, 2000),
    (64, 131, 20001), (65, 512, 513), (100, 65, 4097), (129, 64, 1023), (257, 64, 513),
    (515, 777, 1030), (2100, 100, 3001), (2100, 1000, 9000), (70, 1024, 180001),
    (400, 64, (1 << 21) + 77)])
def test_cross_entropy_writes_its_outputs_alone(rows, width, vocab, dtype, rocm_device, ho):
    lib, elem = ho.load_library(), torch.finfo(dtype).bits // 8
    for k, pads in enumerate(((0, 0), (3, 5))):
        hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, vocab, dtype,
                                                       pads=pads)
        tokens[::7] = IGNORE
        what, past = f"[{rows}, {width}, {vocab}] {dtype} {k}", elem * (3 * k)
        sizes = [rows, width, vocab, width + pads[0], width + pads[1], 0.7, IGNORE]
        given = [address(hidden), address(weight), elem, address(tokens), 8]
        asked = (address(weight), elem, rows, width, vocab, width + pads[1])
        loss, lse = ho.linear_cross_entropy(hidden, weight, tokens, scale=0.7)
        fenced_call(ho, lib.hipo_linear_cross_entropy, what, (loss, lse), given, sizes,
                    lib.hipo_linear_cross_entropy_workspace_bytes(*asked), rocm_device, 4 * k)
        for two_parts, fn, bytes_of in (
                (False, lib.hipo_linear_cross_entropy_bwd,
                 lib.hipo_linear_cross_entropy_bwd_workspace_bytes),
                (True, lib.hipo_linear_cross_entropy_bwd_two_parts,
                 lib.hipo_linear_cross_entropy_bwd_two_parts_workspace_bytes)):
            got = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse, scale=0.7,
                                              grad_lse=grads[1], two_parts=two_parts)
            fenced_call(ho, fn, f"{what} gradient {two_parts}", got,
                        [address(grads[0]), *given, address(lse), address(grads[1])], sizes,
                        bytes_of(*asked), rocm_device, past)


# ---------------------------------------------------------------------------
# Pieces of the gradients, row strides far above the width, every call of a run
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [*LAYERS, (2100, 100, 3001), (2100, 1000, 9000),
                                              (300, 264, 20001), (40, 264, 20001)])
def test_gradients_row_by_row(rows, width, vocab, dtype, rocm_device, ho):
    """Of d = g_lse p with probabilities near one another, so that a piece of d
    that is missing or wrong shows in the 2-norm of a row of dhidden (64 of 2000
    tokens: a sixth of it) and of 64 rows of dweight, whose worst-case bounds
    would hide it.  bf16: half a step, 2^-8, of d and of the result.  fp32: ln p,
    below 16, is off by half a step, 2^-21, and so is its product, 2^-20.5; with
    the logits' and the sums' own 2^-19."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, vocab, dtype, std=0.5)
    _, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    zero = torch.zeros_like(lse)
    h, w = hidden.double(), weight.double()
    d = torch.exp(h @ w.t() - lse[:, None].double()) * grads[1][:, None].double()
    want = d @ w, d.t() @ h
    least = 2.0 ** -7 if dtype == BF16 else 2.0 ** -18
    for two_parts in (False, True):
        got = ho.linear_cross_entropy_bwd(zero, hidden, weight, tokens, lse, grad_lse=grads[1],
                                          two_parts=two_parts)
        for name, u, v, strip in zip(("dhidden", "dweight"), got, want, (1, 64)):
            for first in range(0, len(v), strip * 4096):
                some = slice(first, first + strip * 4096)
                off, size = ((u.double() - v)[some], v[some])
                off, size = (torch.stack([p.norm() for p in t.split(strip)]) if strip > 1
                             else t.norm(dim=-1) for t in (off, size))
                worst = float((off / size).max())
                assert worst <= least, f"[{rows}, {width}, {vocab}] {dtype} {name}: {worst:.2e}"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab,more", [(3, 65, 300, 9), (5, 72, 1000, 0),
                                                   (40, 72, 300, 0), (100, 72, 300, 0),
                                                   (260, 264, 600, 0), (100, 72, 300, 8)])
def test_row_strides_far_above_the_width(rows, width, vocab, more, dtype, rocm_device, ho):
    """Up to the largest of the weight, 2^21, and past 2^31 bytes of hidden."""
    pads = (2 ** 31 // (2 * rows) + 5 + more - width, 2 ** 21 - more - width)
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, vocab, dtype,
                                                   pads=pads)
    assert weight.stride(0) == 2 ** 21 - more and hidden.stride(0) * rows * 2 > 2 ** 31
    got = ho.linear_cross_entropy(hidden, weight, tokens)
    near = [t.contiguous() for t in (hidden, weight)]
    check_loss(ho, *near, tokens, grads, f"[{rows}, {width}, {vocab}] {dtype}")
    for k, (u, (v, tol)) in enumerate(zip(got, ref.linear_cross_entropy(*near, tokens))):
        ref.close(u, v, tol, f"[{rows}, {width}, {vocab}] {dtype} {k}")
    lse = got[1]
    for two_parts in (False, True):
        kw = dict(grad_lse=grads[1], two_parts=two_parts)
        a = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse, **kw)
        wanted = ref.linear_cross_entropy_bwd(grads[0], *near, tokens, lse, grad_lse=grads[1])
        for name, u, (v, tol) in zip(("dhidden", "dweight"), a, wanted):
            ref.close(u, v, tol, f"[{rows}, {width}, {vocab}] {dtype} {name}")


class Checked:
    """The library, each call's results held to the 64-bit formulas of the
    operands that it had."""

    def __init__(self, ho):
        self.ho, self.calls = ho, 0
        self.embedding, self.embedding_bwd = ho.embedding, ho.embedding_bwd

    def close(self, names, got, want):
        self.calls += 1
        for name, u, v in zip(names, got, want):
            if v is not None:
                ref.close(u, v[0].cpu(), v[1].cpu(), f"call {self.calls} {name}")

    def block_norms(self, x, residual, **kw):
        h, y, stats = self.ho.block_norms(x, residual, **kw)
        want_h, tol_h, _, _ = ref.stream(x, residual, **kw)
        want_y, tol_y, _, _ = ref.after(h, **kw)
        self.close(("h", "y"), (h, y), ((want_h, tol_h), (want_y, tol_y)))
        return h, y, stats

    def block_norms_bwd(self, *args, **kw):
        got = self.ho.block_norms_bwd(*args, **kw)
        self.close(("dx", "dresidual", "dgate", "dpost", "dpost_bias", "dpre", "dpre_bias"), got,
                   ref.block_norms_bwd(*args, **kw))
        return got

    def linear_cross_entropy(self, *args, scale):
        got = self.ho.linear_cross_entropy(*args, scale=scale)
        self.close(("loss", "lse"), got, ref.linear_cross_entropy(*args, scale))
        return got

    def linear_cross_entropy_bwd(self, *args, scale):
        got = self.ho.linear_cross_entropy_bwd(*args, scale=scale)
        self.close(("dhidden", "dweight"), got, ref.linear_cross_entropy_bwd(*args, scale))
        return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [(40, 64, 300), (260, 520, 2003), (2100, 264, 5001)])
def test_every_call_of_a_run(rows, width, vocab, dtype, rocm_device, ho):
    """What a run's roundings between its calls would hide."""
    checked = Checked(ho)
    Model(checked, rocm_device, rows, width, vocab, dtype).step()
    assert checked.calls == 6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width,vocab", [(3, 20, 300), (20, 72, 20001), (50, 72, 300),
                                              (100, 72, 700), (2100, 100, 33000)])
def test_infinite_logits(rows, width, vocab, dtype, rocm_device, ho):
    """-infinity adds nothing and is a loss of +infinity for its own token;
    dhidden is NaN in the columns where 0 is multiplied with an infinite weight
    and as without that token in the others, and dweight is finite."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, width, vocab, dtype)
    hidden = hidden.abs() + 0.125  # (no 0, and all of one sign)
    weight = weight.clone()
    gone = [0, vocab // 2, vocab - 1]
    weight[gone, 7] = -INF
    tokens = torch.where(torch.isin(tokens, torch.tensor(gone, device=rocm_device)), 1, tokens)
    tokens[1] = gone[1]
    got = ho.linear_cross_entropy(hidden, weight, tokens)
    left = torch.ones(vocab, dtype=torch.bool, device=rocm_device)
    left[gone] = False
    place = torch.cumsum(left, 0) - 1
    there = torch.where(torch.arange(rows, device=rocm_device) == 1, -1, place[tokens])
    assert got[0][1] == INF and torch.isfinite(got[1]).all()
    wanted = ref.linear_cross_entropy(hidden, weight[left], there)
    for name, u, (v, tol) in zip(("loss", "lse"), got, wanted):
        u = u.clone()
        u[1], v[1] = (0.0, 0.0) if name == "loss" else (u[1], v[1])
        ref.close(u, v, tol, f"[{rows}, {width}, {vocab}] {dtype} {name}")
    tokens[1] = 1
    dh, dw = ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, got[1])
    want = ref.linear_cross_entropy_bwd(grads[0], hidden, weight[left], place[tokens], got[1])
    rest = [c for c in range(width) if c != 7]
    assert dh[:, 7].isnan().all()
    ref.close(dh[:, rest], want[0][0][:, rest], want[0][1][:, rest], f"{rows} {dtype} dhidden")
    ref.close(dw[left], *want[1], f"{rows} {dtype} dweight")
    assert not dw[gone].any()
    weight[vocab // 3, 7] = INF
    got = ho.linear_cross_entropy(hidden, weight, tokens)
    assert not torch.isfinite(got[1]).any() and not torch.isfinite(got[0]).any()


@pytest.mark.parametrize("rows", [3, 70, 300, 2500])
@pytest.mark.parametrize("kind", ["some", "all", "but one", "unknown", "nan"])
def test_two_parts_of_rows_left_out(kind, rows, rocm_device, ho):
    """Rows of ignore_index count nowhere, whatever they hold; NaN where one part
    has NaN, and the others' values near those of one part."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, rows, 72, 600, BF16)
    out = torch.zeros(rows, dtype=torch.bool, device=rocm_device)
    if kind == "some":
        out[::3] = True
    elif kind in ("all", "but one"):
        out[:] = True
        out[rows // 2] = kind == "all"
    tokens[out] = IGNORE
    hidden[out] = NAN
    if kind == "unknown":
        tokens[0], tokens[rows // 2] = 600, -1
    if kind == "nan":
        hidden[rows // 2, 5] = NAN
    _, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    one, two = (ho.linear_cross_entropy_bwd(grads[0], hidden, weight, tokens, lse,
                                            grad_lse=grads[1], two_parts=k) for k in (False, True))
    for u, v in zip(one, two):
        assert torch.equal(u.isnan(), v.isnan())
        fine = ~u.isnan()
        assert float((u - v)[fine].double().norm()) <= 2.0 ** -7 * float(u[fine].double().norm())
    assert not two[0][out].any()
    if kind in ("unknown", "nan"):
        assert two[0][rows // 2].isnan().all() and two[1].isnan().all()
    if kind == "all":
        assert not two[1].any()


def test_two_parts_in_a_graph(rocm_device, ho):
    """Replayed on new tokens, another number of them left out, with eager work
    between."""
    hidden, weight, tokens, grads = layer_operands(rocm_device, 300, 264, 2003, BF16)
    lse = torch.full_like(grads[0], 9.0)
    call = lambda: ho.linear_cross_entropy_bwd(  # noqa: E731
        grads[0], hidden, weight, tokens, lse, grad_lse=grads[1], two_parts=True)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        captured = call()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        tokens.copy_(torch.randint(0, 2003, (300,), generator=g))
        tokens[:seed * 100] = IGNORE
        eager = [v.clone() for v in call()]
        graph.replay()
        torch.cuda.synchronize()
        for u, v in zip(captured, eager):
            assert torch.equal(u, v), f"replay {seed}"


# ---------------------------------------------------------------------------
# Offsets past 32 bits
# ---------------------------------------------------------------------------

def normal(dev, *shape, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    t = torch.empty(*shape, dtype=BF16, device=dev)
    for part in t.split(1 << 18):
        part.normal_(0.0, std, generator=g)
    return t


@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_norms_of_more_rows_than_workgroups(norm, rocm_device, ho):
    """2^20 workgroups of one row each and a few rows more, of 4.3e9 values: the
    rows are as in a call of their own."""
    rows, cols = (1 << 20) + 5, 4099
    x, r, gh, gy = (normal(rocm_device, rows, cols, seed=k) for k in range(4))
    w, v = (normal(rocm_device, cols, seed=k) for k in (5, 6))
    kw = dict(post=w, pre=v, gate=w, norm=norm, scale=0.5, offset=1.0)
    h, y, stats = ho.block_norms(x, r, **kw)
    got = ho.block_norms_bwd(gh, gy, x, h, stats, **kw)
    assert all(torch.isfinite(t).all() for t in got[2:] if t is not None)
    for some in (slice(0, 9), slice(rows // 2, rows // 2 + 9), slice(rows - 9, rows)):
        part = [t[some].contiguous() for t in (x, r, gh, gy)]
        for u, own in zip((h, y, stats), ho.block_norms(*part[:2], **kw)):
            assert torch.equal(u[some], own)
        own = ho.block_norms_bwd(*part[2:], part[0], h[some].contiguous(),
                                 stats[some].contiguous(), **kw)
        assert torch.equal(got[0][some], own[0]) and torch.equal(got[1][some], own[1])


@pytest.mark.parametrize("rows", [3, 70])
def test_output_layers_of_more_than_32_bits(rows, rocm_device, ho):
    """A weight and its gradient of 4.3e9 values, in the kernels of few rows and in
    the products; d = g_lse p, every row of the weight counting about as much."""
    width, vocab = 2056, (1 << 21) + 100
    weight = normal(rocm_device, vocab, width, std=0.5 / width ** 0.5)
    hidden = normal(rocm_device, rows, width, seed=1)
    tokens = torch.linspace(0, vocab - 1, rows, device=rocm_device).round().long()
    loss, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    h = hidden.double()
    s = torch.cat([h @ w.double().t() for w in weight.split(1 << 17)], 1)
    want = torch.logsumexp(s, -1)
    # Of values below 16: a few steps of 2^-20.
    assert float((lse - want).abs().max()) < 2.0 ** -17
    assert float((loss - (want - s.gather(1, tokens[:, None])[:, 0])).abs().max()) < 2.0 ** -17
    one, zero = torch.ones_like(lse), torch.zeros_like(lse)
    p = torch.exp(s - lse.double()[:, None])
    dh_want = sum(q @ w.double() for q, w in zip(p.split(1 << 17, 1), weight.split(1 << 17)))
    for two_parts in (False, True):
        dh, dw = ho.linear_cross_entropy_bwd(zero, hidden, weight, tokens, lse, grad_lse=one,
                                             two_parts=two_parts)
        off = (dh.double() - dh_want).norm(dim=-1) / dh_want.norm(dim=-1)
        assert float(off.max()) <= 2.0 ** -7
        for some in (slice(0, 300), slice(vocab // 2, vocab // 2 + 300), slice(vocab - 300, vocab)):
            v = p[:, some].t() @ h
            off = (dw[some].double() - v).norm(dim=-1) / v.norm(dim=-1)
            assert float(off.max()) <= 2.0 ** -7, some


def test_hidden_states_of_more_than_32_bits(rocm_device, ho):
    """4.3e9 values of hidden and dhidden: rows as in a call of their own, to what
    other tiles' sums may differ by."""
    rows, width, vocab = (1 << 22) - 256, 1032, 70
    hidden = normal(rocm_device, rows, width)
    weight = normal(rocm_device, vocab, width, seed=1, std=0.5 / width ** 0.5)
    tokens = torch.arange(rows, device=rocm_device) % vocab
    tokens[::5] = IGNORE
    loss, lse = ho.linear_cross_entropy(hidden, weight, tokens)
    grad = torch.ones(rows, device=rocm_device)
    dh, dw = ho.linear_cross_entropy_bwd(grad, hidden, weight, tokens, lse)
    assert torch.isfinite(dw).all() and torch.isfinite(loss).all()
    for some in (slice(0, 500), slice(rows // 2, rows // 2 + 500), slice(rows - 500, rows)):
        args = (hidden[some], weight, tokens[some])
        for u, (v, tol) in zip((loss, lse), ref.linear_cross_entropy(*args)):
            ref.close(u[some], v, tol, f"{some}")
        v, tol = ref.linear_cross_entropy_bwd(grad[some], *args, lse[some])[0]
        ref.close(dh[some], v, tol, f"{some} dhidden")
