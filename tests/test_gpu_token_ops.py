"""Token log probabilities, embeddings and their gradients on the GPU against
the 64-bit reference, at the sizes, masks, types and strides where they could
go wrong; refusals; streams, graphs and a run of all of them together."""
import pytest
import torch

import token_ops_reference as ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NAN, INF, IGNORE = ref.NAN, ref.INF, ref.IGNORE
DTYPES = [BF16, F32]


@pytest.fixture(scope="module")
def ho():
    import hip_oracles
    hip_oracles.load_library()
    return hip_oracles


def strided(x, dev, pad, shift):
    """x on the device as rows of a buffer of NaN, `pad` values between rows,
    `shift` values off the buffer's start."""
    rows, cols = x.shape
    buf = torch.full((rows * (cols + pad) + shift,), NAN, dtype=x.dtype, device=dev)
    view = buf[shift:].view(rows, cols + pad)[:, :cols]
    view.copy_(x)
    return view


def make_logits(rows, vocab, dtype, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 3
    if kind == "ties":       # few distinct values
        x = torch.randint(-3, 4, (rows, vocab), generator=g).float()
        x[torch.rand(rows, vocab, generator=g) < 0.1] = -0.0
    elif kind == "equal":
        x = torch.full((rows, vocab), 1.5)
    elif kind == "rising":
        x = torch.arange(vocab).float().expand(rows, vocab) * 1e-3
    elif kind == "falling":
        x = -torch.arange(vocab).float().expand(rows, vocab) * 1e-3
    elif kind == "masked":   # one in ten is left; the first row keeps one place
        x[torch.rand(rows, vocab, generator=g) < 0.9] = -INF
        x[0] = -INF
        x[0, vocab // 2] = 0.25
    elif kind == "peaked":
        x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] = 60.0
    elif kind == "special":  # rows of their own: nothing left, lowest, infinite, NaN
        x = x.to(dtype).float()
        low = torch.finfo(dtype).min
        x[0] = -INF
        x[1 % rows] = low
        if rows > 2:
            x[2] = low
            x[2, vocab // 3] = 1.0
        if rows > 3:
            x[3, vocab - 1] = INF
        if rows > 4:
            x[4, vocab // 2] = NAN
        if rows > 5:
            x[5, 0] = -INF
        if rows > 6:  # far apart, of both signs
            x[6] = low
            x[6, vocab // 4] = -low
    x = x.to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g)
    return x, t


def check_forward(ho, dev, x, t, *, scale=1.0, top=0, pad=0, shift=0, wide=True, what=""):
    xd = strided(x, dev, pad, shift)
    td = t.to(torch.int64 if wide else torch.int32).to(dev)
    got = ho.token_logprobs(xd, td, scale=scale, entropy=True, top=top)
    torch.cuda.synchronize()
    (lp, lse, ent, tv, ti), (tol_lp, tol_lse, tol_h, tol_top) = ref.token_logprobs(
        x, t, scale, top=top)
    ref.close(got[0], lp, tol_lp, f"{what} logprob")
    ref.close(got[1], lse, tol_lse, f"{what} lse")
    ref.close(got[2], ent, tol_h, f"{what} entropy")
    if top:
        assert torch.equal(got[4].cpu(), ti), f"{what} top ids"
        ref.close(got[3], tv, tol_top, f"{what} top")
    plain = ho.token_logprobs(xd, td, scale=scale)
    assert len(plain) == 2
    for a, b in zip(plain, got):  # the options change nothing else
        assert torch.equal(a.isnan(), b.isnan())
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)), what


SHAPES = [(1, 1), (1, 7), (3, 8), (7, 64), (5, 1000), (2, 8191), (9, 8192), (3, 50001),
          (64, 1024), (700, 517), (1, 131072), (2, 262147), (1100, 4097)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_forward_sizes(rows, vocab, dtype, rocm_device, ho):
    x, t = make_logits(rows, vocab, dtype, "plain", rows + vocab)
    for k, top in enumerate((0, 1, 20, 64)):
        check_forward(ho, rocm_device, x, t, top=min(top, vocab), scale=(1.0, 0.7)[k % 2],
                      pad=(0, 3, 8, 0)[k], shift=(0, 1, 8, 5)[k], wide=k % 2 == 0,
                      what=f"[{rows}, {vocab}] {dtype} top {top}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["ties", "equal", "rising", "falling", "masked", "peaked",
                                  "special"])
def test_forward_values(kind, dtype, rocm_device, ho):
    for rows, vocab in ((8, 33), (8, 3000), (9, 40007), (600, 2500), (1, 200000), (8, 100003)):
        x, t = make_logits(rows, vocab, dtype, kind, 11)
        if kind == "masked":
            t[0] = vocab // 2
        for top in (5, 33):
            check_forward(ho, rocm_device, x, t, top=top, scale=0.5 if top == 5 else 1.25,
                          shift=3 * (top == 5), what=f"{kind} [{rows}, {vocab}] {dtype} top {top}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(6, 100), (6, 70001), (1030, 3001)])
def test_forward_ignored_and_unknown_tokens(rows, vocab, dtype, rocm_device, ho):
    x, t = make_logits(rows, vocab, dtype, "plain", 5)
    t[0], t[1], t[2], t[3] = IGNORE, -1, vocab, vocab - 1
    x[0] = NAN  # not read
    check_forward(ho, rocm_device, x, t, top=9, what="tokens")
    t[:] = IGNORE
    check_forward(ho, rocm_device, x, t, top=9, wide=False, what="all ignored")
    t[:] = torch.randint(0, vocab, (rows,))
    x[0] = 0.5
    td, xd = t.to(rocm_device), x.to(rocm_device)
    got = ho.token_logprobs(xd, td, ignore_index=int(t[4]), top=2)
    assert (got[0][t == t[4]] == 0).all() and (got[3][t.to(rocm_device) == t[4]] == -1).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [
    (511, 2049), (1023, 4100), (1024, 4096), (1024, 8200), (300, 2048), (128, 24600), (129, 24600),
    (127, 49160), (129, 49152), (256, 32000), (257, 32003), (5, 49151), (40, 60001)])
def test_forward_where_the_workgroups_change(rows, vocab, dtype, rocm_device, ho):
    x, t = make_logits(rows, vocab, dtype, "plain", vocab - rows)
    check_forward(ho, rocm_device, x, t, top=3, shift=rows % 2, what=f"[{rows}, {vocab}] {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(2, 4096), (3, 30000), (130, 32768), (2, 131072)])
def test_alternatives_that_a_few_lanes_hold(rows, vocab, dtype, rocm_device, ho):
    """Every second run of 32 16-byte vectors far above the others: the largest
    of 64 lanes' values say little."""
    g = torch.Generator().manual_seed(vocab)
    run = 32 * 16 // dtype.itemsize
    x = torch.randn(rows, vocab, generator=g) + 50.0 * ((torch.arange(vocab) // run) % 2)
    t = torch.randint(0, vocab, (rows,), generator=g)
    for top in (20, 33, 64):
        check_forward(ho, rocm_device, x.to(dtype), t, top=top, what=f"stripes {vocab} {top}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(14, 40), (14, 3000), (14, 66000), (1100, 2100)])
def test_logits_far_from_zero(rows, vocab, dtype, rocm_device, ho):
    """Rows of nothing but a mask value, logits around large numbers, maxima that
    rise past where the statistics change their form (c x = 2^20)."""
    g = torch.Generator().manual_seed(vocab)
    at = [-1e4, -65504.0, -1e6, -1e9, -1e10, -1e20, -1e30, 3e5, 1e6, 5e7, -7.2e5, 726000.0, 1e5]
    x = torch.randn(rows, vocab, generator=g) * 3
    for r in range(len(at)):
        x[r] = at[r] if r in (3, 4, 5, 6) else at[r] + x[r]
    x[11] += torch.arange(vocab) * (3000.0 / vocab)
    x[12, vocab // 2] = 9e5   # near, then far
    x[13, :vocab // 2] = -1e9
    t = torch.randint(0, vocab, (rows,), generator=g)
    for scale in (1.0, 0.7):
        check_forward(ho, rocm_device, x.to(dtype), t, scale=scale, top=4,
                      what=f"far [{rows}, {vocab}] {dtype} {scale}")


@pytest.mark.parametrize("rows,vocab", [(4, 5000), (3, 70000)])
def test_alternatives_where_one_number_fills_the_row(rows, vocab, rocm_device, ho):
    """fp32 logits that no bf16 value is near: a mask of -1e9 with fewer places
    left than alternatives asked for, the rest ties."""
    x = torch.full((rows, vocab), -1e9)
    x[:, 7::vocab // 5] = torch.randn(rows, len(range(7, vocab, vocab // 5)))
    check_forward(ho, rocm_device, x, torch.full((rows,), 7), top=20, what="masked by -1e9")


def test_forward_is_the_same_alone_and_in_a_batch_of_its_kind(rocm_device, ho):
    x, t = make_logits(300, 9001, BF16, "plain", 8)
    xd, td = x.to(rocm_device), t.to(rocm_device)
    a = ho.token_logprobs(xd, td, entropy=True, top=8)
    b = ho.token_logprobs(xd, td, entropy=True, top=8)
    for u, v in zip(a, b):
        assert torch.equal(u, v)


def bwd_inputs(rows, vocab, dtype, kind, seed):
    x, t = make_logits(rows, vocab, dtype, kind, seed)
    g = torch.Generator().manual_seed(seed + 1)
    if kind == "masked":
        t[0] = vocab // 2
    grads = [torch.randn(rows, generator=g) for _ in range(3)]
    (_, lse, ent, _, _), _ = ref.token_logprobs(x, torch.zeros(rows, dtype=torch.int64))
    return x, t, grads, lse, ent


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,kind", [
    (1, 1, "plain"), (3, 7, "plain"), (5, 64, "plain"), (4, 1000, "masked"), (3, 8191, "plain"),
    (2, 50001, "plain"), (1, 131072, "peaked"), (700, 517, "plain"), (7, 4099, "ties"),
    (9, 16384, "masked"), (5, 2049, "plain"), (6, 2945, "ties"), (3, 4100, "masked"),
    (4, 6145, "plain")])
def test_backward(rows, vocab, kind, dtype, rocm_device, ho):
    x, t, (g, gh, gl), _, _ = bwd_inputs(rows, vocab, dtype, kind, rows + vocab)
    for k, (use_h, use_l) in enumerate(((0, 0), (1, 0), (0, 1), (1, 1))):
        scale = (1.0, 0.7, 1.0, 1.25)[k]
        (_, lse, ent, _, _), _ = ref.token_logprobs(x, torch.zeros(rows, dtype=torch.int64), scale)
        lse, ent = lse.float(), ent.float()
        if rows > 2 and k == 3:
            t[0], t[1] = IGNORE, vocab
            lse[0] = 0.0
        kw = dict(scale=scale, entropy=ent if use_h else None, grad_entropy=gh if use_h else None,
                  grad_lse=gl if use_l else None)
        want, tol = ref.token_logprobs_bwd(g, x, t, lse, **kw)
        dev = {a: v.to(rocm_device) if isinstance(v, torch.Tensor) else v for a, v in kw.items()}
        xd = strided(x, rocm_device, (0, 3, 8, 0)[k], (0, 1, 0, 5)[k])
        td = t.to(rocm_device).to(torch.int32 if k % 2 else torch.int64)
        got = ho.token_logprobs_bwd(g.to(rocm_device), xd, td, lse.to(rocm_device), **dev)
        ref.close(got, want, tol, f"[{rows}, {vocab}] {kind} {dtype} {k}")
        # Into rows with gaps, which stay; then in place.
        pad = 5
        out = torch.full((rows, vocab + pad), 7.0, dtype=dtype, device=rocm_device)
        r = ho.token_logprobs_bwd(g.to(rocm_device), xd, td, lse.to(rocm_device),
                                  out=out[:, :vocab], **dev)
        assert r.data_ptr() == out.data_ptr()
        assert torch.equal(out[:, :vocab].isnan(), got.isnan())
        assert torch.equal(out[:, :vocab].nan_to_num(3.0), got.nan_to_num(3.0))
        assert (out[:, vocab:] == 7.0).all()
        ho.token_logprobs_bwd(g.to(rocm_device), xd, td, lse.to(rocm_device), out=xd, **dev)
        assert torch.equal(xd.nan_to_num(3.0), got.nan_to_num(3.0))


def test_backward_of_rows_that_are_left_out_or_not_finite(rocm_device, ho):
    x, t = make_logits(8, 3001, BF16, "special", 2)
    (_, lse, _, _, _), _ = ref.token_logprobs(x, t)
    t[4] = IGNORE  # the NaN row
    g = torch.ones(8)
    got = ho.token_logprobs_bwd(*(v.to(rocm_device) for v in (g, x, t, lse.float()))).cpu()
    assert (got[4] == 0).all()
    assert got[0].isnan().all() and torch.isfinite(got[[1, 2, 5, 6, 7]]).all()
    t[:] = IGNORE
    got = ho.token_logprobs_bwd(*(v.to(rocm_device) for v in (g, x, t, lse.float()))).cpu()
    assert (got == 0).all()


def test_forward_results_feed_the_backward(rocm_device, ho):
    """The kernel's own lse and entropy, and the gradient against differences
    of the 64-bit forward."""
    rows, vocab, scale, h = 4, 40, 0.7, 1e-4
    x, t = make_logits(rows, vocab, F32, "plain", 9)
    gs = [torch.randn(rows) for _ in range(3)]
    d = [v.to(rocm_device) for v in (x, t, *gs)]
    lp, lse, ent = ho.token_logprobs(d[0], d[1], scale=scale, entropy=True)
    got = ho.token_logprobs_bwd(d[2], d[0], d[1], lse, scale=scale, entropy=ent,
                                grad_entropy=d[3], grad_lse=d[4]).double().cpu()

    def loss(x):
        (lp, lse, ent, _, _), _ = ref.token_logprobs(x, t, scale)
        return gs[0] * lp + gs[1] * ent + gs[2] * lse

    want = torch.empty(rows, vocab, dtype=torch.float64)
    for j in range(vocab):
        e = torch.zeros(rows, vocab, dtype=torch.float64)
        e[:, j] = h
        want[:, j] = (loss(x.double() + e) - loss(x.double() - e)) / (2 * h)
    # h^2 times a third derivative (below 100 here: |x| <= 12), and fp32 of
    # values below 40: lse and entropy off by a few 2^-24 * 40.
    assert float((got - want).abs().max()) < 100 * h * h + 64 * ref.U * 40


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,width,vocab", [
    ((), 64, 10), ((1,), 1, 1), ((5,), 7, 20), ((3, 4), 1001, 50), ((16,), 2048, 300),
    ((1000,), 8, 70000), ((33,), 4096, 5), ((70001,), 12, 9), ((2, 3, 5), 8193, 11)])
def test_embedding(shape, width, vocab, dtype, rocm_device, ho):
    g = torch.Generator().manual_seed(width)
    w = torch.randn(vocab, width, generator=g).to(dtype)
    t = torch.randint(0, vocab, shape, generator=g)
    for k, scale in enumerate((1.0, 0.7, 64.0)):
        if k == 2 and t.numel() > 2:
            t.view(-1)[0], t.view(-1)[1], t.view(-1)[2] = -1, vocab, vocab - 1
        wd = strided(w, rocm_device, (0, 3, 8)[k], (0, 1, 0)[k])
        td = t.to(rocm_device).to(torch.int32 if k % 2 else torch.int64)
        got = ho.embedding(wd, td, scale=scale)
        assert got.shape == (*shape, width) and got.dtype == dtype
        known = (t >= 0) & (t < vocab)
        want = (w.float()[torch.where(known, t, 0)] * scale).to(dtype)
        want[~known] = NAN
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(3.0), want.nan_to_num(3.0))
        exact = ref.embedding(w, t, scale)
        tol = (ref.HALF[dtype] + ref.U * 1.01) * exact.abs() + 2.0 ** -126
        ref.close(got, exact, tol, f"{shape} {width} {dtype}")


def ids_of(kind, count, vocab, g):
    if kind == "uniform":
        return torch.randint(0, vocab, (count,), generator=g)
    if kind == "one":
        return torch.full((count,), vocab - 1)
    if kind == "text":  # a few ids make up much of it
        u = torch.rand(count, generator=g).double()
        return ((vocab + 1.0) ** u).floor().long().sub(1).clamp(0, vocab - 1)
    if kind == "runs":
        return torch.arange(count) // 7 % vocab
    t = torch.randint(0, vocab, (count,), generator=g)  # "unknown": some outside
    t[::3] = torch.tensor([-1, vocab, vocab + 5, -100])[torch.arange(len(t[::3])) % 4]
    return t


def test_ids_past_32_bits(rocm_device, ho):
    """int64 ids whose lower half alone would be one of the vocabulary."""
    far = torch.tensor([3 + (1 << 32), 3 - (1 << 32), 2, 3 + (1 << 40), 3])
    x, _ = make_logits(5, 50, F32, "plain", 1)
    lp = ho.token_logprobs(x.to(rocm_device), far.to(rocm_device))[0].cpu()
    assert lp.isnan().tolist() == [True, True, False, True, False]
    w = torch.randn(50, 8, device=rocm_device)
    e = ho.embedding(w, far.to(rocm_device))
    assert e.isnan().all(-1).tolist() == [True, True, False, True, False]
    dw = ho.embedding_bwd(torch.ones(5, 8, device=rocm_device), far.to(rocm_device), 50)
    assert dw[2].eq(1).all() and dw[3].eq(1).all() and float(dw.sum()) == 16.0


@pytest.mark.parametrize("dtype,out", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16)])
@pytest.mark.parametrize("count,width,vocab,kind", [
    (0, 64, 50, "uniform"), (1, 1, 1, "one"), (1, 64, 1000, "uniform"), (7, 5, 3, "uniform"),
    (64, 96, 64, "runs"), (65, 768, 3000, "text"), (1000, 1001, 517, "text"),
    (4096, 40, 50001, "text"), (5000, 264, 70, "uniform"), (20000, 16, 3, "uniform"),
    (70001, 8, 1025, "text"), (3000, 2048, 11, "one"), (9000, 8, 2000, "one"),
    (300, 4096, 100, "unknown"), (2049, 33, 131073, "uniform"), (16, 8, 2, "one"), (17, 8, 2, "one"),
    (1024, 512, 3000, "text"), (1024, 513, 3000, "text"), (1025, 16, 3000, "text"),
    (1023, 100, 7, "uniform"), (513, 700, 40, "one"), (1000, 5, 300, "unknown"),
    (16, 32769, 5, "text"), (16, 32768, 5, "text"), (32, 24, 1, "one"), (33, 24, 1, "one"),
    (64, 24, 2, "one"), (96, 24, 3, "runs"), (16384, 24, 9000, "text"),
    (17, 94, 13054, "text"), (900, 3, 20011, "text"), (300, 1, 70001, "uniform"),
    (33000, 8, 300000, "text"), (8193, 64, 8192, "runs")])
def test_embedding_backward(count, width, vocab, kind, dtype, out, rocm_device, ho):
    g = torch.Generator().manual_seed(count + width)
    t = ids_of(kind, count, vocab, g)
    grad = torch.randn(count, width, generator=g).to(dtype)
    what = f"{count} x {width} into {vocab} {kind} {dtype} {out}"
    for k, scale in enumerate((1.0, 0.7)):
        pad = None if k == 0 or count == 0 else max(0, min(vocab - 1, int(t[0])))
        gd = grad.to(rocm_device)
        td = t.to(rocm_device).to(torch.int32 if k else torch.int64)
        want, tol, touched = ref.embedding_bwd(grad, t, vocab, scale, pad, dtype=out)
        got = ho.embedding_bwd(gd, td, vocab, scale=scale, padding_idx=pad, dtype=out)
        assert got.dtype == out
        ref.close(got, want, tol, what)
        assert (got.cpu()[~touched] == 0).all()
        again = ho.embedding_bwd(gd, td, vocab, scale=scale, padding_idx=pad, dtype=out)
        assert torch.equal(got, again), f"{what}: two calls differ"
        base = torch.randn(vocab, width, generator=g).to(out)
        base[~touched] = NAN  # neither read for a sum nor written
        buf = base.to(rocm_device)
        r = ho.embedding_bwd(gd, td, vocab, scale=scale, padding_idx=pad, into=buf)
        assert r is buf
        want, tol, _ = ref.embedding_bwd(grad, t, vocab, scale, pad, into=base, dtype=out)
        ref.close(buf[touched], want[touched], tol[touched], f"{what} into")
        assert buf.cpu()[~touched].isnan().all()


@pytest.mark.parametrize("count", [500, 1500])  # without and with a sort
def test_embedding_backward_keeps_what_lies_behind(count, rocm_device, ho):
    """Rows of an odd width at the end of a larger buffer."""
    width, vocab = 37, 41
    g = torch.Generator().manual_seed(1)
    t = ids_of("text", count, vocab, g).to(rocm_device)
    grad = torch.randn(count, width, generator=g).to(BF16).to(rocm_device)
    for out in DTYPES:
        buf = torch.full((vocab * width + 64,), 5.0, dtype=out, device=rocm_device)
        ho.embedding_bwd(grad, t, vocab, into=buf[:vocab * width].view(vocab, width))
        assert (buf[vocab * width:] == 5.0).all()


def test_refusals(rocm_device, ho):
    dev = rocm_device
    x = torch.zeros(4, 16, dtype=BF16, device=dev)
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    f = torch.zeros(4, device=dev)
    bad = [
        lambda: ho.token_logprobs(x.half(), t), lambda: ho.token_logprobs(x[0], t),
        lambda: ho.token_logprobs(x, t.float()), lambda: ho.token_logprobs(x, t[:3]),
        lambda: ho.token_logprobs(x.t().contiguous().t(), t),
        lambda: ho.token_logprobs(x[:1].expand(4, 16), t),
        lambda: ho.token_logprobs(x, t, scale=0.0), lambda: ho.token_logprobs(x, t, scale=INF),
        lambda: ho.token_logprobs(x, t, top=17), lambda: ho.token_logprobs(x, t, top=-1),
        lambda: ho.token_logprobs(x, torch.zeros(8, dtype=torch.int64, device=dev)[::2]),
        lambda: ho.token_logprobs(x, t.cpu()),
        lambda: ho.token_logprobs(x[:, :0], t),
        lambda: ho.token_logprobs_bwd(f.double(), x, t, f),
        lambda: ho.token_logprobs_bwd(f[:3], x, t, f), lambda: ho.token_logprobs_bwd(f, x, t, f[:3]),
        lambda: ho.token_logprobs_bwd(f, x, t, f, grad_entropy=f),
        lambda: ho.token_logprobs_bwd(f, x, t, f, out=torch.zeros(4, 16, device=dev)),
        lambda: ho.token_logprobs_bwd(f, x, t, f, out=x[:1].expand(4, 16)),
        lambda: ho.token_logprobs_bwd(f, x, t, f, out=x[:, :8]),
        lambda: ho.token_logprobs_bwd(f, x.view(-1)[:32].view(4, 8), t, f,
                                      out=x.view(-1)[:64].view(4, 16)[:, :8]),
        lambda: ho.token_logprobs_bwd(f, x.view(-1)[:32].view(4, 8), t, f,
                                      out=x.view(-1)[1:33].view(4, 8)),
        lambda: ho.token_logprobs_bwd(f, x[:, :8], t, f, out=x[:, 4:12]),
        lambda: ho.embedding(x.half(), t), lambda: ho.embedding(x, t.float()),
        lambda: ho.embedding(x.t(), t), lambda: ho.embedding(x[0], t),
        lambda: ho.embedding(x[:1].expand(4, 16), t),
        lambda: ho.embedding_bwd(x.half(), t, 9), lambda: ho.embedding_bwd(x[:3], t, 9),
        lambda: ho.embedding_bwd(x.t(), t, 9), lambda: ho.embedding_bwd(x, t, -1),
        lambda: ho.embedding_bwd(x, t, 9, dtype=torch.float16),
        lambda: ho.embedding_bwd(x, t, 9, padding_idx=9),
        lambda: ho.embedding_bwd(x, t, 9, padding_idx=-1),
        lambda: ho.embedding_bwd(x, t, 9, into=torch.zeros(8, 16, device=dev)),
        lambda: ho.embedding_bwd(x, t, 9, into=torch.zeros(16, 9, device=dev).t()),
        lambda: ho.embedding_bwd(x, t, 9, dtype=BF16, into=torch.zeros(9, 16, device=dev)),
        lambda: ho.embedding_bwd(x, t, 4, into=x),
        lambda: ho.embedding_bwd(x, t, 3, into=x[1:]),
    ]
    for k, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            print(f"refusal {k} was not one")


def test_backward_into_other_columns_of_the_logits_buffer(rocm_device, ho):
    x, t = make_logits(6, 200, F32, "plain", 4)
    buf = torch.zeros(6, 400, device=rocm_device)
    buf[:, :200] = x.to(rocm_device)
    g = torch.ones(6, device=rocm_device)
    _, lse = ho.token_logprobs(buf[:, :200], t.to(rocm_device))
    want = ho.token_logprobs_bwd(g, x.to(rocm_device), t.to(rocm_device), lse)
    ho.token_logprobs_bwd(g, buf[:, :200], t.to(rocm_device), lse, out=buf[:, 200:])
    assert torch.equal(buf[:, 200:], want) and torch.equal(buf[:, :200].cpu(), x)


def test_empty_calls(rocm_device, ho):
    t = torch.zeros(0, dtype=torch.int64, device=rocm_device)
    x = torch.zeros(0, 16, device=rocm_device)
    outs = ho.token_logprobs(x, t, entropy=True, top=3)
    assert [tuple(o.shape) for o in outs] == [(0,), (0,), (0,), (0, 3), (0, 3)]
    f = torch.zeros(0, device=rocm_device)
    assert ho.token_logprobs_bwd(f, x, t, f).shape == (0, 16)
    assert ho.embedding(torch.zeros(4, 8, device=rocm_device), t).shape == (0, 8)
    assert ho.embedding(torch.zeros(4, 0, device=rocm_device), t + 0).shape == (0, 0)
    dw = ho.embedding_bwd(x, t, 5)
    assert dw.shape == (5, 16) and (dw == 0).all()
    assert ho.embedding_bwd(x, t, 0).shape == (0, 16)


def test_offsets_past_32_bits(rocm_device, ho):
    """Rows that start after 2^31 values, in each operator."""
    rows, vocab = 33, (1 << 26) + 5
    x = torch.empty(rows, vocab, dtype=BF16, device=rocm_device).normal_()
    t = torch.randint(0, vocab, (rows,), device=rocm_device)
    got = ho.token_logprobs(x, t, entropy=True, top=3)
    last = x[-1].double()
    ls = torch.log_softmax(last, -1)
    tol = 2.0 ** -24 * (vocab / 64 / 64 + 512)
    assert abs(float(got[0][-1]) - float(ls[t[-1]])) < tol
    assert abs(float(got[1][-1]) - float(torch.logsumexp(last, -1))) < tol
    best = last.max()
    assert int(got[4][-1, 0]) == int((last == best).nonzero()[0])
    print("offsets: forward", flush=True)
    g = torch.ones(rows, device=rocm_device)
    dx = ho.token_logprobs_bwd(g, x, t, got[1])
    want = -(last - got[1][-1].double()).exp()
    want[t[-1]] += 1
    err = (dx[-1].double() - want).abs()
    assert bool((err <= 2.0 ** -8 * want.abs() * 1.01 + 1e-30).all())
    del x, dx, last, ls, want, err
    print("offsets: backward", flush=True)
    width, vocab = 2048, (1 << 20) + (1 << 16)
    w = torch.empty(vocab, width, dtype=BF16, device=rocm_device).normal_()
    t = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device=rocm_device)
    e = ho.embedding(w, t)
    assert torch.equal(e, w[t])
    dw = ho.embedding_bwd(e, t, vocab)
    assert torch.equal(dw[-1], (2 * e[0].float()).to(BF16)) and torch.equal(dw[-2], e[2])
    assert torch.equal(dw[0], e[1]) and int((dw != 0).any(-1).sum()) == 3
    far = torch.cat([t, torch.full((1100,), -1, device=rocm_device)])  # sorted
    assert torch.equal(ho.embedding_bwd(torch.cat([e, w[:1100]]), far, vocab), dw)
    t = torch.full(((1 << 20) + 9,), 3, dtype=torch.int32, device=rocm_device)
    t[-1] = vocab - 1
    e = ho.embedding(w, t)
    assert torch.equal(e[-1], w[-1]) and torch.equal(e[-2], w[3])
    print("offsets: embedding", flush=True)


def test_other_streams_and_no_change_of_device_state(rocm_device, ho):
    x, t = make_logits(50, 9001, BF16, "plain", 3)
    xd, td = x.to(rocm_device), t.to(rocm_device)
    w = torch.randn(9001, 96, device=rocm_device)
    a = [*ho.token_logprobs(xd, td, top=4), ho.embedding(w, td)]
    many, wide = td.repeat(30), torch.randn(1500, 96, device=rocm_device)
    a += [ho.embedding_bwd(a[-1], td, 9001), ho.embedding_bwd(wide, many, 9001)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):  # two at a time, each with its own workspace
        for s in streams:
            with torch.cuda.stream(s):
                b = [*ho.token_logprobs(xd, td, top=4), ho.embedding(w, td)]
                b += [ho.embedding_bwd(b[-1], td, 9001), ho.embedding_bwd(wide, many, 9001)]
                outs.append(b)
    torch.cuda.synchronize()
    for b in outs:
        for u, v in zip(a, b):
            assert torch.equal(u, v)


class Model:
    """Token ids to their log probabilities through one tied table, and back."""

    def __init__(self, ho, dev, rows, width, vocab, seed):
        g = torch.Generator().manual_seed(seed)
        self.ho, self.vocab, self.width = ho, vocab, width
        self.w = (torch.randn(vocab, width, generator=g)).to(BF16).to(dev)
        self.gamma = (1 + 0.1 * torch.randn(width, generator=g)).to(BF16).to(dev)
        self.ids = torch.randint(0, vocab, (rows,), generator=g).to(dev)
        self.next = torch.randint(0, vocab, (rows,), generator=g).to(dev)
        self.next[::5] = IGNORE
        self.grad = torch.full((rows,), -1.0 / rows, device=dev)

    def step(self):
        ho = self.ho
        h = ho.embedding(self.w, self.ids, scale=self.width ** 0.5)
        y = ho.rmsnorm_ex(h, self.gamma, 1e-6, mode=1, scale=self.width ** -0.5)
        logits = y @ self.w.t()
        logprob, lse, ent, tv, ti = ho.token_logprobs(logits, self.next, entropy=True, top=4)
        dl = ho.token_logprobs_bwd(self.grad, logits, self.next, lse, entropy=ent,
                                   grad_entropy=0.01 * self.grad)
        dw = (dl.t() @ y).float()          # the head's part of the tied gradient
        dy = dl @ self.w                   # stands for what reaches the lookup
        dw = ho.embedding_bwd(dy, self.ids, self.vocab, scale=self.width ** 0.5, into=dw)
        return h, y, logits, logprob, lse, ent, tv, ti, dl, dy, dw


def test_a_run_of_all_of_them(rocm_device, ho):
    m = Model(ho, rocm_device, 200, 256, 3001, 1)
    h, y, logits, logprob, lse, ent, tv, ti, dl, dy, dw = m.step()
    assert torch.equal(h, (m.w[m.ids].float() * 16.0).to(BF16))
    (rlp, rlse, rent, rtv, rti), (a, b, c, d) = ref.token_logprobs(logits, m.next, top=4)
    ref.close(logprob, rlp, a, "logprob")
    ref.close(lse, rlse, b, "lse")
    ref.close(ent, rent, c, "entropy")
    ref.close(tv, rtv, d, "top")
    assert torch.equal(ti.cpu(), rti)
    want, tol = ref.token_logprobs_bwd(m.grad, logits, m.next, lse, entropy=ent,
                                       grad_entropy=0.01 * m.grad)
    ref.close(dl, want, tol, "dlogits")
    head = (dl.t() @ y).float()
    want, tol, _ = ref.embedding_bwd(dy, m.ids, m.vocab, 16.0, into=head)
    ref.close(dw, want, tol, "tied gradient")


@pytest.mark.parametrize("rows", [120, 1100])
def test_the_run_in_a_graph(rows, rocm_device, ho):
    """Captured once and replayed on new tokens, with eager work between."""
    m = Model(ho, rocm_device, rows, 128, 2003, 2)
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
        if seed == 2:
            m.ids.fill_(7)
        eager = [v.clone() for v in m.step()]
        graph.replay()
        torch.cuda.synchronize()
        for k, (u, v) in enumerate(zip(captured, eager)):
            assert torch.equal(u, v), f"replay {seed}, output {k}"


def test_embedding_backward_into_the_largest_vocabulary(rocm_device, ho):
    """2^30 rows, 36 GB of gradient: the most workgroups that sort beside the
    most that write zeros."""
    width, vocab = 17, 1 << 30
    t = torch.tensor([vocab - 1, 0, 1 << 29, vocab - 1], device=rocm_device)
    grad = torch.randn(4, width, device=rocm_device).to(BF16)
    dw = ho.embedding_bwd(grad, t, vocab)
    torch.cuda.synchronize()
    print("largest vocabulary: launched", flush=True)
    assert torch.equal(dw[0], grad[1]) and torch.equal(dw[1 << 29], grad[2])
    assert torch.equal(dw[-1], (grad[0].float() + grad[3].float()).to(BF16))
    dw[t] = 0
    flat = dw.view(-1)
    assert not any(bool(part.any()) for part in flat.split(1 << 30))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(2, 4096), (3, 30000), (130, 32768), (2, 131072)])
def test_alternatives_that_a_few_lanes_hold_with_nan(rows, vocab, dtype, rocm_device, ho):
    """As above, and the first value, whose key is the largest there is, is NaN;
    then others too."""
    g = torch.Generator().manual_seed(vocab)
    run = 32 * 16 // dtype.itemsize
    x = torch.randn(rows, vocab, generator=g)
    t = torch.randint(0, vocab, (rows,), generator=g)
    for high in (0, 1):
        y = (x + 50.0 * ((torch.arange(vocab) // run + high) % 2)).to(dtype)
        y[:, 0] = NAN
        for top in (1, 33, 34, 64):
            check_forward(ho, rocm_device, y, t, top=top, what=f"stripes {vocab} {top} {high}")
        y[1:, ::run] = NAN
        check_forward(ho, rocm_device, y, t, top=64, what=f"stripes {vocab} {high}, more NaN")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [
    (40, 70), (64, 2001), (1100, 4097), (300, 9001), (40, 33000), (6, 262147), (2048, 8200)])
@pytest.mark.parametrize("scale", [1.0, 0.7, 1.25])
def test_no_probability_above_one(rows, vocab, scale, dtype, rocm_device, ho):
    """Rows that one token decides, alone or 17 to 30 above 200 others: no log
    probability above 0, no entropy below, lse not below the largest value; of
    a token that is alone exactly 0."""
    g = torch.Generator().manual_seed(vocab)
    t = torch.randint(0, vocab, (rows,), generator=g)
    high = torch.randn(rows, generator=g) * 30.0
    high[::20] *= 1e5  # far from zero too
    x = torch.full((rows, vocab), -INF)
    for r in range(1, rows, 2):
        others = torch.randint(0, vocab, (200,), generator=g)
        x[r, others] = high[r] - 17.0 - r % 14 + torch.randn(200, generator=g)
    x[torch.arange(rows), t] = high
    x = x.to(dtype)
    lp, lse, ent, tv, _ = (v.cpu() for v in ho.token_logprobs(
        x.to(rocm_device), t.to(rocm_device), scale=scale, entropy=True, top=3))
    assert (lp <= 0).all() and (tv <= 0).all()
    assert (ent >= 0).all()
    largest = x.double().amax(-1) * float(torch.tensor(scale))
    assert (lse >= largest.float()).all()
    assert (lp[::2] == 0).all() and (ent[::2] == 0).all()


def test_a_gradient_over_its_other_inputs_is_refused(rocm_device, ho):
    """fp32 vectors, and tokens, in the memory that the gradient is written to."""
    rows, vocab = 4, 16
    x = torch.zeros(rows, vocab, device=rocm_device)
    t = torch.zeros(rows, dtype=torch.int64, device=rocm_device)
    f = torch.zeros(rows, device=rocm_device)
    out = torch.zeros(rows, 2 * vocab, device=rocm_device)
    inside, between = out[1, 4:8], out[1, vocab:vocab + rows]
    ids = out[0, :2 * rows].view(torch.int64)
    for kw in (dict(grad=inside), dict(lse=inside), dict(tokens=ids),
               dict(entropy=inside, grad_entropy=f), dict(entropy=f, grad_entropy=inside),
               dict(grad_lse=inside), dict(lse=out[0, vocab - 1:vocab + 3])):
        with pytest.raises(ValueError, match="overlaps"):
            ho.token_logprobs_bwd(**{"grad": f, "logits": x, "tokens": t, "lse": f,
                                     "out": out[:, :vocab], **kw})
    # Between the rows there is room.
    f += 2.0
    between.copy_(f)
    got = ho.token_logprobs_bwd(f, x, t, between, out=out[:, :vocab])
    assert torch.equal(got, ho.token_logprobs_bwd(f, x, t, f)) and (between == 2.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("rows,vocab", [(2048, 8200), (2049, 16421), (2500, 50001)])
def test_forward_of_many_long_rows(rows, vocab, shift, dtype, rocm_device, ho):
    """The kernel of a training batch, with and without each option; every 61st
    row against the reference, ignored and unknown tokens among them."""
    g = torch.Generator(device=rocm_device).manual_seed(vocab)
    buf = torch.empty(rows * (vocab + 3) + shift, dtype=dtype, device=rocm_device)
    x = buf[shift:].view(rows, vocab + 3)[:, :vocab]
    x.copy_(torch.randn(rows, vocab, generator=g, device=rocm_device) * 3)
    t = torch.randint(0, vocab, (rows,), generator=g, device=rocm_device)
    some = torch.arange(0, rows, 61, device=rocm_device)
    t[some[1]], t[some[2]], x[some[1]] = IGNORE, vocab, NAN
    x[some[3], :vocab // 2] = -INF
    want, tol = ref.token_logprobs(x[some], t[some], 0.7, top=3)
    for top in (0, 3):
        for entropy in (False, True):
            got = list(ho.token_logprobs(x, t, scale=0.7, entropy=entropy, top=top))
            torch.cuda.synchronize()
            what = f"[{rows}, {vocab}] {dtype} top {top} entropy {entropy}"
            if not entropy:
                got.insert(2, None)
            for k in range(3 + (top > 0)):
                if got[k] is not None:
                    ref.close(got[k][some], want[k], tol[k], f"{what} {k}")
            if top:
                assert torch.equal(got[4][some].cpu(), want[4]), what


def test_rows_do_not_depend_on_their_batch(rocm_device, ho):
    """A row has the same bits in other batches of the same plan wherever it
    begins at the same place of 16 bytes.  (Its values are added by the 16-byte
    vectors that they lie in: elsewhere in another order, within the bound.)"""
    for rows, vocab, part in ((300, 9001, slice(7, 270)), (1500, 700, slice(100, 1300)),
                              (60, 50001, slice(3, 61)), (100, 9000, slice(11, 12))):
        for dtype in DTYPES:
            x, t = make_logits(rows, vocab, dtype, "plain", rows)
            xd, td = x.to(rocm_device), t.to(rocm_device)
            begins = (torch.arange(rows) * vocab * dtype.itemsize) % 16
            whole = ho.token_logprobs(xd, td, entropy=True, top=8)
            order = torch.randperm(rows, generator=torch.Generator().manual_seed(1))
            want, tol = ref.token_logprobs(x, t, top=8)
            for some in (torch.arange(rows)[part], order):
                what = f"[{rows}, {vocab}] {dtype}"
                got = ho.token_logprobs(xd[some], td[some], entropy=True, top=8)
                same = begins[some] == begins[:len(some)]
                assert bool(same.any()) or some is not order, what
                for k, (u, v) in enumerate(zip(whole, got)):
                    assert torch.equal(u[some][same], v[same]), f"{what}: bits"
                    if k < 4:
                        ref.close(v, want[k][some], tol[k][some], what)
                assert torch.equal(got[4].cpu(), want[4][some]), what
            # The same rows where they are.
            for u, v in zip(whole, ho.token_logprobs(xd[part], td[part], entropy=True, top=8)):
                assert torch.equal(u[part], v), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(49153, 9), (100000, 17), (98305, 700)])
def test_backward_of_more_rows_than_a_grid_layer(rows, vocab, dtype, rocm_device, ho):
    x, t = make_logits(rows, vocab, dtype, "plain", vocab)
    t[::7], t[5::11] = IGNORE, -1
    x[::14] = NAN  # ignored
    g = torch.Generator().manual_seed(rows)
    grads = [torch.randn(rows, generator=g) for _ in range(3)]
    (_, lse, ent, _, _), _ = ref.token_logprobs(x, t)
    lse, ent = lse.float(), ent.float()
    kw = dict(entropy=ent, grad_entropy=grads[1], grad_lse=grads[2])
    want, tol = ref.token_logprobs_bwd(grads[0], x, t, lse, **kw)
    dev = {k: v.to(rocm_device) for k, v in kw.items()}
    got = ho.token_logprobs_bwd(*(v.to(rocm_device) for v in (grads[0], x, t, lse)), **dev)
    ref.close(got, want, tol, f"[{rows}, {vocab}] {dtype}")


def test_more_rows_than_a_launch(rocm_device, ho):
    """2^23 workgroups in a launch of the forward, 2^30 lanes in one of the
    lookup and of the embedding gradient: the rest in launches of their own."""
    g = torch.Generator(device=rocm_device).manual_seed(1)
    rows, vocab = (1 << 23) + 1001, 5
    x = torch.randn(rows, vocab, generator=g, device=rocm_device)
    t = torch.randint(0, vocab, (rows,), generator=g, device=rocm_device)
    lp, lse, best, which = ho.token_logprobs(x, t, top=1)
    ls = torch.log_softmax(x.double(), -1)
    # |x| < 8: a few halves of a step of numbers below 16.
    tol = 16 * 16 * ref.U
    assert float((lp - ls.gather(1, t[:, None])[:, 0]).abs().max()) < tol
    assert float((lse - torch.logsumexp(x.double(), -1)).abs().max()) < tol
    assert torch.equal(which[:, 0], x.argmax(-1))
    assert float((best - ls.amax(-1, keepdim=True)).abs().max()) < tol
    del x, t, lp, lse, best, which, ls
    print("launches: forward", flush=True)
    count = (1 << 30) + 1001
    w = torch.randn(7, 1, generator=g, device=rocm_device)
    t = torch.arange(count, dtype=torch.int32, device=rocm_device) % 7
    e = ho.embedding(w, t)
    for part in range(0, count, 1 << 28):
        some = slice(part, part + (1 << 28))
        assert torch.equal(e[some], w[t[some].long()])
    del t, e
    print("launches: embedding", flush=True)
    count, width, vocab = 40000, 1 << 18, 3
    t = torch.randint(0, vocab, (count,), generator=g, device=rocm_device)
    t[-1000:] = vocab  # adds nothing
    grad = torch.empty(count, width, dtype=BF16, device=rocm_device).normal_(generator=g)
    dw = ho.embedding_bwd(grad, t, vocab, dtype=F32)
    for cols in (slice(0, 9), slice(width // 2 - 4, width // 2 + 4), slice(width - 9, width)):
        want, tol, _ = ref.embedding_bwd(grad[:, cols], t, vocab)
        ref.close(dw[:, cols], want, tol, f"columns {cols}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 130, 256])
def test_forward_where_the_threads_of_a_row_change(rows, dtype, rocm_device, ho):
    """Three and four rounds of 256 threads' loads, and a value less and more."""
    values = 256 * 4 * 16 // dtype.itemsize
    for vocab in (2 * values + 1, 3 * values - 1, 3 * values + 16 // dtype.itemsize,
                  4 * values - 1, 4 * values + 1):
        x, t = make_logits(rows, vocab, dtype, "plain", vocab)
        check_forward(ho, rocm_device, x, t, top=20, shift=1, what=f"[{rows}, {vocab}] {dtype}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_of_rows_with_infinities(dtype, rocm_device, ho):
    """As its description says: NaN rows with NaN or with nothing left, and the
    place of a +inf."""
    x, t = make_logits(9, 2100, dtype, "special", 3)
    t[:] = 7
    xd, td = x.to(rocm_device), t.to(rocm_device)
    g = torch.ones(9, device=rocm_device)
    _, lse = ho.token_logprobs(xd, td)
    got = ho.token_logprobs_bwd(g, xd, td, lse).cpu()
    assert got[0].isnan().all() and got[4].isnan().all()
    assert got[3].isnan().nonzero()[:, 0].tolist() == [2099] and got[3, 7] == 1
    assert torch.isfinite(got[[1, 2, 5, 6, 7, 8]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("power", [-100, -40, 100])
@pytest.mark.parametrize("rows,vocab", [(40, 700), (300, 9001), (6, 100003)])
def test_scales_that_are_powers_of_two(rows, vocab, power, dtype, rocm_device, ho):
    """Logits and a scale that cancel are the logits with scale 1, bit by bit;
    the gradient is that times the scale, but for what is below 2^-126."""
    x, t = make_logits(rows, vocab, dtype, "masked", 6)
    t[0] = vocab // 2
    xd, td = x.to(rocm_device), t.to(rocm_device)
    far = xd * 2.0 ** -power
    assert torch.equal(far.float() * 2.0 ** power, xd.float())
    one = ho.token_logprobs(xd, td, entropy=True, top=5)
    got = ho.token_logprobs(far, td, scale=2.0 ** power, entropy=True, top=5)
    for u, v in zip(one, got):
        assert torch.equal(u, v)
    g = torch.randn(3, rows, generator=torch.Generator().manual_seed(1)).to(rocm_device)
    kw = dict(entropy=one[2], grad_entropy=g[1], grad_lse=g[2])
    want = ho.token_logprobs_bwd(g[0], xd, td, one[1], **kw).double() * 2.0 ** power
    dx = ho.token_logprobs_bwd(g[0], far, td, one[1], scale=2.0 ** power, **kw).double()
    normal = want.abs() >= 2.0 ** -125
    assert torch.equal(dx[normal], want[normal])
    assert float((dx - want)[~normal].abs().max()) <= 2.0 ** -126
