"""Token log probabilities and embeddings without a GPU: argument checks of the
entry points, empty calls, and the 64-bit reference against finite differences
and torch's own functions."""
import pytest
import torch

import hip_oracles
import token_ops_reference as ref

HIPO_EINVAL = 1000
P = 16  # a pointer that no call here reads


@pytest.fixture(scope="module")
def lib():
    return hip_oracles.load_library()


def fwd(lib, *, x=P, es=2, tok=P, ts=8, lp=P, lse=P, ent=None, tv=None, ti=None, rows=2, vocab=8,
        stride=8, scale=1.0, top=0, ws=None, wb=0):
    return lib.hipo_token_logprobs(x, es, tok, ts, lp, lse, ent, tv, ti, rows, vocab, stride,
                                   scale, -100, top, ws, wb, None)


def bwd(lib, *, g=P, x=P, es=2, tok=P, ts=8, lse=P, ent=None, ge=None, gl=None, dx=32, rows=2,
        vocab=8, stride=8, dstride=8, scale=1.0):
    return lib.hipo_token_logprobs_bwd(g, x, es, tok, ts, lse, ent, ge, gl, dx, rows, vocab,
                                       stride, dstride, scale, -100, None)


def emb(lib, *, w=P, es=2, tok=P, ts=8, out=P, n=2, d=8, v=8, stride=8):
    return lib.hipo_embedding(w, es, tok, ts, out, n, d, v, stride, 1.0, None)


def emb_bwd(lib, *, g=P, es=2, tok=P, ts=8, dw=P, os=2, n=2, d=8, v=8, pad=-1, acc=0, ws=P,
            wb=1 << 40):
    return lib.hipo_embedding_bwd(g, es, tok, ts, dw, os, n, d, v, 1.0, pad, acc, ws, wb, None)


@pytest.mark.parametrize("call,kw,msg", [
    (fwd, dict(rows=-1), b"negative"), (fwd, dict(es=3), b"elem_size"),
    (fwd, dict(ts=2), b"token_size"), (fwd, dict(scale=0.0), b"scale"),
    (fwd, dict(scale=-1.0), b"scale"), (fwd, dict(scale=float("inf")), b"scale"),
    (fwd, dict(scale=float("nan")), b"scale"), (fwd, dict(stride=7), b"row_stride"),
    (fwd, dict(top=9), b"top"), (fwd, dict(top=-1), b"top"),
    (fwd, dict(vocab=100, stride=100, top=65), b"top"),
    (fwd, dict(vocab=0, stride=0), b"empty vocabulary"), (fwd, dict(x=None), b"null"),
    (fwd, dict(tok=None), b"null"), (fwd, dict(lp=None), b"null"), (fwd, dict(lse=None), b"null"),
    (fwd, dict(top=2), b"null"), (fwd, dict(vocab=1 << 31, stride=1 << 31), b"2^31"),
    (fwd, dict(rows=1 << 31), b"2^31"),
    (bwd, dict(rows=-1), b"negative"), (bwd, dict(es=8), b"elem_size"),
    (bwd, dict(ts=1), b"token_size"), (bwd, dict(scale=0.0), b"scale"),
    (bwd, dict(stride=7), b"row_stride"), (bwd, dict(dstride=7), b"row_stride"),
    (bwd, dict(ge=P), b"entropy"), (bwd, dict(dx=P, dstride=9), b"in place"),
    (bwd, dict(g=None), b"null"), (bwd, dict(dx=None), b"null"), (bwd, dict(lse=None), b"null"),
    (bwd, dict(vocab=1 << 31, stride=1 << 31, dstride=1 << 31), b"2^31"),
    (emb, dict(n=-1), b"negative"), (emb, dict(es=1), b"elem_size"),
    (emb, dict(ts=16), b"token_size"), (emb, dict(stride=7), b"row_stride"),
    (emb, dict(v=0), b"empty vocabulary"), (emb, dict(w=None), b"null"),
    (emb, dict(out=None), b"null"), (emb, dict(n=1 << 31), b"2^31"),
    (emb_bwd, dict(n=-1), b"negative"), (emb_bwd, dict(es=1), b"elem_size"),
    (emb_bwd, dict(os=8), b"out_size"), (emb_bwd, dict(ts=0), b"token_size"),
    (emb_bwd, dict(g=None), b"null"), (emb_bwd, dict(dw=None), b"null"),
    (emb_bwd, dict(tok=None), b"null"), (emb_bwd, dict(v=1 << 31), b"2^31"),
])
def test_arguments_are_checked_before_any_launch(lib, call, kw, msg):
    assert call(lib, **kw) == HIPO_EINVAL
    assert msg in lib.hipo_last_error()


def test_workspaces_are_checked(lib):
    need = lib.hipo_token_logprobs_workspace_bytes(1, 1 << 20, 8)
    if need:
        kw = dict(rows=1, vocab=1 << 20, stride=1 << 20, top=8, tv=P, ti=P)
        assert fwd(lib, **kw, ws=P, wb=need - 1) == HIPO_EINVAL
        assert b"workspace" in lib.hipo_last_error()
        assert fwd(lib, **kw, ws=None, wb=need) == HIPO_EINVAL
        assert b"workspace" in lib.hipo_last_error()
        assert fwd(lib, **kw, ws=8, wb=need) == HIPO_EINVAL
        assert b"workspace" in lib.hipo_last_error()
    need = lib.hipo_embedding_bwd_workspace_bytes(4096, 768, 32000)
    if need:
        kw = dict(n=4096, d=768, v=32000)
        for ws, wb in ((P, need - 1), (None, need), (8, need)):
            assert emb_bwd(lib, **kw, ws=ws, wb=wb) == HIPO_EINVAL
            assert b"workspace" in lib.hipo_last_error()
    assert lib.hipo_token_logprobs_workspace_bytes(0, 100, 0) == 0
    assert lib.hipo_embedding_bwd_workspace_bytes(1024, 512, 32000) == 0  # no sort
    assert lib.hipo_embedding_bwd_workspace_bytes(1024, 513, 32000) > 0
    assert lib.hipo_embedding_bwd_workspace_bytes(1025, 8, 32000) > 0
    assert lib.hipo_embedding_bwd_workspace_bytes(1, 16, 1 << 30) == 0
    assert lib.hipo_embedding_bwd_workspace_bytes(1, 17, 1 << 30) > 0


def test_empty_calls_are_no_ops(lib):
    assert fwd(lib, rows=0, x=None, tok=None, lp=None, lse=None) == 0
    assert bwd(lib, rows=0, g=None, x=None, tok=None, lse=None, dx=None) == 0
    assert bwd(lib, vocab=0, stride=0, dstride=0, dx=None) == 0
    assert emb(lib, n=0, w=None, tok=None, out=None) == 0
    assert emb(lib, d=0, w=None, tok=None, out=None) == 0
    assert emb_bwd(lib, v=0, g=None, tok=None, dw=None) == 0
    assert emb_bwd(lib, d=0, g=None, tok=None, dw=None) == 0
    assert lib.hipo_last_error() == b""


def test_wrappers_refuse_cpu_tensors():
    x, t = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: hip_oracles.token_logprobs(x, t),
                 lambda: hip_oracles.token_logprobs_bwd(x[:, 0], x, t, x[:, 0]),
                 lambda: hip_oracles.embedding(x, t),
                 lambda: hip_oracles.embedding_bwd(x, t, 8)):
        with pytest.raises(ValueError, match="ROCm device only"):
            call()


def test_reference_against_torch_functions():
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 37, generator=g) * 3
    x[2, 5:] = -ref.INF
    t = torch.tensor([0, 36, 4, ref.IGNORE, 9])
    (lp, lse, ent, top, ids), _ = ref.token_logprobs(x, t, 0.5, top=4)
    ls = torch.log_softmax(x.double() * 0.5, -1)
    keep = [0, 1, 2, 4]
    assert torch.allclose(lp[keep], ls[keep, t[keep]], atol=1e-12)
    assert torch.allclose(lse[keep], torch.logsumexp(x.double() * 0.5, -1)[keep], atol=1e-12)
    assert torch.allclose(ent[keep], torch.special.entr(ls.exp()).sum(-1)[keep], atol=1e-12)
    assert torch.allclose(top[keep], ls[keep].gather(1, ids[keep]), atol=1e-12)
    assert (lp[3], lse[3], ent[3]) == (0, 0, 0) and (ids[3] == -1).all()


@pytest.mark.parametrize("scale", [1.0, 0.7])
def test_reference_gradient_against_differences(scale):
    g = torch.Generator().manual_seed(4)
    rows, vocab, h = 3, 11, 1e-4
    x = torch.randn(rows, vocab, generator=g).double()
    t = torch.randint(0, vocab, (rows,), generator=g)
    gs = [torch.randn(rows, generator=g).double() for _ in range(3)]

    def loss(x):
        (lp, lse, ent, _, _), _ = ref.token_logprobs(x, t, scale)
        return gs[0] * lp + gs[1] * ent + gs[2] * lse

    (_, lse, ent, _, _), _ = ref.token_logprobs(x, t, scale)
    got, _ = ref.token_logprobs_bwd(gs[0], x.float(), t, lse, scale, entropy=ent,
                                    grad_entropy=gs[1], grad_lse=gs[2])
    want = torch.empty_like(x)
    for j in range(vocab):
        e = torch.zeros_like(x)
        e[:, j] = h
        want[:, j] = (loss(x + e) - loss(x - e)) / (2 * h)
    # Differences are off by about h^2 times a third derivative; x is rounded to
    # fp32 for the formula.
    assert torch.allclose(got, want, atol=3e-6)


def test_reference_embedding_gradient_against_differences():
    g = torch.Generator().manual_seed(5)
    w = torch.randn(6, 3, generator=g)
    t = torch.tensor([[1, 4, 4], [0, 1, 4]])
    go = torch.randn(2, 3, 3, generator=g)
    got, _, touched = ref.embedding_bwd(go, t, 6, 1.5)
    wd = w.double().requires_grad_()
    (torch.nn.functional.embedding(t, wd) * 1.5 * go.double()).sum().backward()
    assert torch.allclose(got, wd.grad, atol=1e-12)
    assert touched.tolist() == [True, True, False, False, True, False]


@pytest.mark.parametrize("dtype", [torch.float32, torch.int64])
def test_vectors_beside_rows_of_a_buffer(dtype):
    """Every place of a vector in and about rows with a gap, against the bytes."""
    stride, cols, rows = 12, 7, 3
    buf = torch.zeros(64, dtype=torch.bfloat16)
    a = buf[8:8 + rows * stride].view(rows, stride)[:, :cols]
    held = torch.zeros(64, dtype=torch.bool)
    held[8:8 + rows * stride].view(rows, stride)[:, :cols] = True
    step = dtype.itemsize // 2
    for at in range(0, 64, step):
        for n in range(0, (64 - at) // step + 1):
            t = buf[at:at + n * step].view(dtype)
            want = not bool(held[at:at + n * step].any())
            assert hip_oracles._apart_from_rows(t, a, stride, rows, cols) == want, (at, n)


def test_workspaces_are_needed_where_rows_or_tokens_are_split():
    """What the sizes' checks above stand on."""
    lib = hip_oracles.load_library()
    for rows, vocab, top in ((1, 1 << 20, 8), (1, 1 << 20, 0), (64, 128000, 20)):
        assert lib.hipo_token_logprobs_workspace_bytes(rows, vocab, top) > 0
    assert lib.hipo_token_logprobs_workspace_bytes(2048, 8200, 3) == 0
    assert lib.hipo_embedding_bwd_workspace_bytes(4096, 768, 32000) >= 4096 * 16
