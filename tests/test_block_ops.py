"""The norms around a block and the output layer's cross entropy without a GPU:
argument checks of the entry points, empty calls, launches, and the 64-bit
reference against automatic differentiation and differences."""
import re
import subprocess

import numpy as np
import pytest
import torch

import block_ops_reference as ref
import fp32_parts_reference as parts
import hip_oracles
from conftest import ROOT

HIPO_EINVAL = 1000
P = 16  # a pointer that no call here reads
F64 = torch.float64


@pytest.fixture(scope="module")
def lib():
    return hip_oracles.load_library()


def norms(lib, *, x=P, res=P, es=2, post=P, pb=None, pre=P, rb=None, gate=None, h=P, y=P, st=P,
          rows=4, cols=8, gates=0, scale=1.0, offset=0.0, eps=1e-6, layer=0):
    return lib.hipo_block_norms(x, res, es, post, pb, pre, rb, gate, h, y, st, rows, cols, gates,
                                scale, offset, eps, layer, None)


def norms_bwd(lib, *, gh=P, gy=P, x=P, h=P, st=P, es=2, post=P, pb=None, pre=P, rb=None, gate=None,
              dx=P, dr=P, dg=None, dpost=P, dpb=None, dpre=P, drb=None, rows=4, cols=8, gates=0,
              scale=1.0, offset=0.0, layer=0, ws=P, wb=1 << 40):
    return lib.hipo_block_norms_bwd(gh, gy, x, h, st, es, post, pb, pre, rb, gate, dx, dr, dg,
                                    dpost, dpb, dpre, drb, rows, cols, gates, scale, offset, layer,
                                    ws, wb, None)


def loss(lib, *, h=P, w=P, es=2, tok=P, ts=8, out=P, lse=P, rows=2, width=8, vocab=8, hs=8, ws=8,
         scale=1.0, wk=P, wb=1 << 50):
    return lib.hipo_linear_cross_entropy(h, w, es, tok, ts, out, lse, rows, width, vocab, hs, ws,
                                         scale, -100, wk, wb, None)


def loss_bwd(lib, *, g=P, h=P, w=P, es=2, tok=P, ts=8, lse=P, gl=None, dh=P, dw=P, rows=2, width=8,
             vocab=8, hs=8, ws=8, scale=1.0, wk=P, wb=1 << 50):
    return lib.hipo_linear_cross_entropy_bwd(g, h, w, es, tok, ts, lse, gl, dh, dw, rows, width,
                                             vocab, hs, ws, scale, -100, wk, wb, None)


INF, NAN = float("inf"), float("nan")
SIZES = [(dict(es=3), b"elem_size"), (dict(rows=-1), b"negative"), (dict(cols=7), b"cols"),
         (dict(cols=16385), b"cols"), (dict(rows=1 << 31), b"2^31"), (dict(layer=2), b"layer"),
         (dict(scale=INF), b"finite"), (dict(offset=NAN), b"finite"),
         (dict(gate=P), b"gate"), (dict(gates=2), b"gate"), (dict(gates=-1), b"negative")]
LAYER = [(dict(ts=2), b"token_size"), (dict(es=1), b"elem_size"), (dict(rows=-1), b"negative"),
         (dict(vocab=0), b"empty"), (dict(width=0), b"width"), (dict(hs=7), b"row_stride"),
         (dict(ws=7), b"row_stride"), (dict(scale=0.0), b"scale"), (dict(scale=NAN), b"scale"),
         (dict(scale=-1.0), b"scale"), (dict(rows=(1 << 22) - 255), b"2^22"),
         (dict(vocab=1 << 31), b"2^31"), (dict(ws=(1 << 21) + 8), b"2^21"),
         (dict(width=(1 << 20) + 1, hs=1 << 21, ws=1 << 21), b"width"),
         (dict(rows=1 << 19, width=1 << 20, hs=1 << 20, ws=1 << 20), b"2^38"),
         (dict(h=None), b"null"), (dict(w=None), b"null"), (dict(tok=None), b"null"),
         (dict(lse=None), b"null"), (dict(wk=None), b"workspace"), (dict(wb=8), b"workspace"),
         (dict(wk=8), b"workspace")]


@pytest.mark.parametrize("call,kw,msg", [
    *((norms, kw, msg) for kw, msg in SIZES), *((norms_bwd, kw, msg) for kw, msg in SIZES),
    *((loss, kw, msg) for kw, msg in LAYER), *((loss_bwd, kw, msg) for kw, msg in LAYER),
    (norms, dict(post=None, pre=None), b"norm is needed"),
    (norms, dict(post=None, pb=P, layer=1), b"bias needs"),
    (norms, dict(pre=None, rb=P, layer=1), b"bias needs"), (norms, dict(pb=P), b"LayerNorm"),
    (norms, dict(gate=P, gates=3), b"divide"), (norms, dict(eps=-1.0), b"eps"),
    (norms, dict(eps=NAN), b"eps"), (norms, dict(x=None), b"null"), (norms, dict(res=None), b"null"),
    (norms, dict(h=None), b"null"), (norms, dict(y=None), b"null"), (norms, dict(st=None), b"null"),
    (norms_bwd, dict(gate=P, gates=3, dg=P), b"divide"),
    (norms_bwd, dict(pre=None, dpre=None), b"grad_y"),
    (norms_bwd, dict(pre=None, dpre=None, gy=None, gh=None), b"grad_y"),
    (norms_bwd, dict(dpost=None), b"gradient"), (norms_bwd, dict(dpre=None), b"gradient"),
    (norms_bwd, dict(dpb=P), b"gradient"), (norms_bwd, dict(rb=P, layer=1), b"gradient"),
    (norms_bwd, dict(gate=P, gates=1), b"null"), (norms_bwd, dict(x=None), b"null"),
    (norms_bwd, dict(h=None), b"null"), (norms_bwd, dict(gy=None), b"null"),
    (norms_bwd, dict(st=None), b"null"), (norms_bwd, dict(dx=None), b"null"),
    (norms_bwd, dict(dr=None), b"null"), (norms_bwd, dict(ws=None), b"workspace"),
    (norms_bwd, dict(wb=8), b"workspace"), (norms_bwd, dict(ws=8), b"workspace"),
    (loss, dict(out=None), b"null"), (loss_bwd, dict(g=None), b"null"),
    (loss_bwd, dict(dh=None), b"null"), (loss_bwd, dict(dw=None), b"null"),
])
def test_arguments_are_checked_before_any_launch(lib, call, kw, msg):
    assert call(lib, **kw) == HIPO_EINVAL
    assert msg in lib.hipo_last_error()


def test_empty_calls_are_no_ops(lib):
    assert norms(lib, rows=0, x=None, res=None, h=None, y=None, st=None) == 0
    assert norms_bwd(lib, rows=0, x=None, h=None, dx=None, dr=None, st=None, ws=None) == 0
    assert loss(lib, rows=0, h=None, tok=None, out=None, lse=None, wk=None) == 0
    assert loss_bwd(lib, rows=0, g=None, h=None, dh=None, dw=None, wk=None) == 0
    assert lib.hipo_last_error() == b""
    assert lib.hipo_block_norms_bwd_workspace_bytes(0, 64) == 0
    assert lib.hipo_linear_cross_entropy_workspace_bytes(P, 2, 0, 64, 64, 64) == 0
    assert lib.hipo_linear_cross_entropy_bwd_workspace_bytes(P, 2, 0, 64, 64, 64) == 0


def test_workspaces_stay_small(lib):
    """Beside the copy of hidden, the forward keeps no more than 1 / 256 of the
    logits; the gradient keeps a piece of them."""
    for rows, width, vocab in ((8192, 4096, 128000), (1, 2048, 32000), (4096, 64, 200000)):
        pad = -(-rows // 256) * 256
        fwd = lib.hipo_linear_cross_entropy_workspace_bytes(P, 2, rows, width, vocab, width)
        assert 0 < fwd <= pad * (2 * width + 24 + 8 * (vocab // 256 + 1)) + (1 << 26)
        bwd = lib.hipo_linear_cross_entropy_bwd_workspace_bytes(P, 2, rows, width, vocab, width)
        assert 0 < bwd <= (2 << 30) + 12 * pad * (width + 64)


def test_wrappers_refuse_cpu_tensors():
    x, w = torch.zeros(2, 8), torch.zeros(8)
    t, f = torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for call in (lambda: hip_oracles.block_norms(x, x, pre=w),
                 lambda: hip_oracles.block_norms_bwd(x, x, x, x, torch.zeros(2, 4), pre=w),
                 lambda: hip_oracles.linear_cross_entropy(x, x, t),
                 lambda: hip_oracles.linear_cross_entropy_bwd(f, x, x, t, f)):
        with pytest.raises(ValueError, match="ROCm device only"):
            call()


def test_wrappers_refuse_what_is_no_tensor():
    x, w, f = torch.zeros(2, 8), torch.zeros(8), torch.zeros(2)
    t = torch.zeros(2, dtype=torch.int64)
    for bad in (None, [0.0], 1.0, np.zeros((2, 8))):
        for call in (lambda: hip_oracles.block_norms(bad, x, pre=w),
                     lambda: hip_oracles.block_norms_bwd(x, x, bad, x, torch.zeros(2, 4), pre=w),
                     lambda: hip_oracles.linear_cross_entropy(bad, x, t),
                     lambda: hip_oracles.linear_cross_entropy_bwd(f, x, bad, t, f),
                     lambda: hip_oracles.embedding(bad, t),
                     lambda: hip_oracles.row_mean(bad)):
            with pytest.raises(ValueError):
                call()


# ---------------------------------------------------------------------------
# Launches
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    program = tmp_path_factory.mktemp("recorder") / "block_launch_recorder"
    subprocess.run(["g++", "-std=c++17", "-O1", "-rdynamic",
                    str(ROOT / "tests" / "block_launch_recorder.cpp"), str(hip_oracles.LIB_PATH),
                    f"-Wl,-rpath,{hip_oracles.LIB_PATH.parent}", "-Wl,--allow-shlib-undefined",
                    "-o", str(program)], check=True, capture_output=True)

    def run(*calls):
        """([(kernel, grid, block)], return code) of each (FAIL, op, number...)."""
        text = "".join(" ".join(map(str, c)) + "\n" for c in calls)
        out = subprocess.run([str(program)], input=text, check=True, capture_output=True,
                             text=True).stdout.splitlines()
        results, made = [], []
        for line in out:
            m = line.split()
            if m[0] == "rc":
                results.append((made, int(m[1])))
                made = []
            else:
                made.append((m[0], tuple(map(int, m[1:4])), tuple(map(int, m[4:7]))))
        assert len(results) == len(calls)
        return results

    return run


def assert_launchable(made):
    for kernel, grid, block in made:
        assert block[0] * block[1] * block[2] <= 1024, (kernel, block)
        assert grid[1] <= 65535 and grid[2] <= 65535 and min(grid) > 0, (kernel, grid)
        assert all(g * b < 1 << 32 for g, b in zip(grid, block)), (kernel, grid, block)


def test_norms_can_be_launched(launches):
    calls = [(-1, op, rows, cols, gates, elem, layer)
             for op in ("block_norms", "block_norms_bwd") for elem in (2, 4) for layer in (0, 1)
             for rows in (1, 2, 513, 70000, (1 << 31) - 1)
             for cols in (8, 9, 511, 512, 513, 1024, 1025, 2880, 8192, 8193, 16384)
             for gates in (0, 1, rows)]
    for call, (made, rc) in zip(calls, launches(*calls)):
        assert rc == 0 and made, call
        assert_launchable(made)


def test_cross_entropy_can_be_launched(launches):
    sizes = ((1, 1, 1), (1, 2048, 32000), (8192, 4096, 128000), (257, 1001, 50001),
             (5, 8192, 200000), ((1 << 22) - 256, 8, 70000), (3, 8, (1 << 31) - 65536),
             ((1 << 22) - 256, 1 << 16, 300), (3, 1 << 20, 70000))
    calls = [(-1, op, *size, elem) for size in sizes for elem in (2, 4)
             for op in ("linear_cross_entropy", "linear_cross_entropy_bwd")]
    for call, (made, rc) in zip(calls, launches(*calls)):
        assert rc == 0 and made, call
        assert_launchable(made)


@pytest.mark.parametrize("call", [
    ("block_norms", 300, 700, 0, 2, 0), ("block_norms_bwd", 300, 700, 1, 2, 0),
    ("linear_cross_entropy", 300, 200, 3000, 2), ("linear_cross_entropy", 3, 200, 3000, 4),
    ("linear_cross_entropy_bwd", 3, 200, 3000, 2), ("linear_cross_entropy_bwd", 40, 201, 3000, 2),
    ("linear_cross_entropy_bwd", 3, 200, 3000, 4),
    ("linear_cross_entropy_bwd", 300, 200, 3000, 2), ("linear_cross_entropy_bwd", 8192, 4096,
                                                      128000, 4)])
def test_a_refused_launch_ends_the_call(call, launches):
    """Each launch reads what the one before writes."""
    (made, rc), = launches((-1, *call))
    assert rc == 0
    for n, (again, rc) in enumerate(launches(*((n, *call) for n in range(len(made))))):
        assert rc == 9 and again == made[:n + 1]


TWO_PARTS = "linear_cross_entropy_bwd_two_parts"


@pytest.mark.parametrize("rows,elem,threads", [(16, 2, (1024, 1024)), (17, 2, (512, 1024)),
                                               (32, 2, (512, 1024)), (33, 2, (512, 512)),
                                               (16, 4, (512, 512)), (32, 4, (512, 512)),
                                               (33, 4, (256, 256))])
def test_groups_of_few_rows_by_the_registers_they_leave(rows, elem, threads, launches):
    """1024 threads leave a lane 128 registers, which the forward of 17 to 32 rows
    does not fit."""
    calls = [(-1, op, rows, 2048, 16000, elem)
             for op in ("linear_cross_entropy", "linear_cross_entropy_bwd")]
    for want, (made, _) in zip(threads, launches(*calls)):
        (_, _, block), = [m for m in made if "thin_logits" in m[0]]
        assert block == (want, 1, 1)


def test_two_parts_can_be_launched(launches):
    sizes = ((1, 1, 1), (65, 1, 1), (8192, 4096, 128000), (257, 1001, 50001),
             ((1 << 22) - 256, 8, 70000), (65, 8, (1 << 31) - 65536),
             ((1 << 22) - 256, 1 << 16, 300), (65, 1 << 20, 70000))
    calls = [(-1, TWO_PARTS, *size, elem) for size in sizes for elem in (2, 4)]
    for call, (made, rc) in zip(calls, launches(*calls)):
        assert rc == 0 and made, call
        assert_launchable(made)


def test_a_refused_launch_of_two_parts_ends_the_call(launches):
    call = (TWO_PARTS, 300, 200, 3000, 2)
    (made, rc), = launches((-1, *call))
    assert rc == 0
    for n, (again, rc) in enumerate(launches(*((n, *call) for n in range(len(made))))):
        assert rc == 9 and again == made[:n + 1]


def test_the_gradient_of_no_rows_is_written(launches):
    calls = [(-1, op, 0, width, vocab, elem)
             for op in ("linear_cross_entropy_bwd", TWO_PARTS) for elem in (2, 4)
             for width, vocab in ((1, 1), (65, 1001), (1 << 20, (1 << 31) - 65536))]
    for call, (made, rc) in zip(calls, launches(*calls)):
        assert rc == 0 and len(made) == 1 and "zero_weight" in made[0][0], call
        assert_launchable(made)
    (made, rc), = launches((0, "linear_cross_entropy_bwd", 0, 8, 8, 2))
    assert rc == 9 and len(made) == 1


def test_two_parts_check_their_arguments(lib):
    def call(es=2, rows=100, wb=1 << 50, g=P, dw=P):
        return lib.hipo_linear_cross_entropy_bwd_two_parts(
            g, P, P, es, P, 8, P, None, P, dw, rows, 8, 8, 8, 8, 1.0, -100, P, wb, None)

    need = lib.hipo_linear_cross_entropy_bwd_two_parts_workspace_bytes
    for kw, msg in ((dict(es=3), b"elem_size"), (dict(rows=-1), b"negative"),
                    (dict(g=None), b"null"), (dict(wb=need(P, 2, 100, 8, 8, 8) - 1),
                                              b"workspace")):
        assert call(**kw) == HIPO_EINVAL
        assert msg in lib.hipo_last_error() and b"_two_parts" in lib.hipo_last_error()
    assert call(rows=0, dw=None) == 0 and need(P, 2, 0, 8, 8, 8) == 0
    one = lib.hipo_linear_cross_entropy_bwd_workspace_bytes
    for rows, elem, more in ((64, 2, False), (65, 2, True), (8192, 2, False), (65, 4, False)):
        # (Of 8192 rows the pieces are smaller.)
        two = need(P, elem, rows, 4096, 32000, 4096)
        assert (two > one(P, elem, rows, 4096, 32000, 4096)) == more or rows == 8192
        assert two <= (2 << 30) + 12 * max(256, rows) * (4096 + 64)


def test_assembly_names_the_registers_that_it_writes():
    """m0 is no operand: a statement that sets it has to say so."""
    found = 0
    for path in sorted((ROOT / "better-benchmark_amd" / "hip_oracles" / "csrc").iterdir()):
        for asm in re.findall(r"asm volatile\s*\((.*?)\);", path.read_text(), re.S):
            if re.search(r"\bs_\w+ m0,", asm):
                found += 1
                assert '"m0"' in asm.rpartition(":")[2], f"{path.name}: {asm}"
    assert found


# ---------------------------------------------------------------------------
# The reference
# ---------------------------------------------------------------------------

def operands(rows, cols, gates, bias, seed=0):
    g = torch.Generator().manual_seed(seed)
    t = {k: torch.randn(rows, cols, generator=g, dtype=F64) for k in ("x", "residual")}
    kw = {k: torch.randn(cols, generator=g, dtype=F64) for k in ("post", "pre")}
    if bias:
        kw |= {k: torch.randn(cols, generator=g, dtype=F64) for k in ("post_bias", "pre_bias")}
    if gates:
        kw["gate"] = torch.randn(gates, cols, generator=g, dtype=F64)
        if gates == 1:
            kw["gate"] = kw["gate"][0]
    return t, kw


@pytest.fixture
def in_64_bits(monkeypatch):
    monkeypatch.setitem(ref.HALF, F64, 2.0 ** -53)


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("gates", [0, 1, 2, 6])
@pytest.mark.parametrize("which", ["both", "post", "pre"])
def test_norms_reference(which, gates, norm, in_64_bits):
    """Values against torch's own norms, gradients against automatic ones and
    against differences."""
    rows, cols, scale, offset, eps = 6, 5, 0.5, 0.25, 0.125
    t, kw = operands(rows, cols, gates, norm == "layer")
    for k in ("pre", "post"):
        if which not in (k, "both"):
            kw.pop(k)
            kw.pop(k + "_bias", None)
    args = dict(kw, norm=norm, scale=scale, offset=offset, eps=eps)

    def forward(x, residual, **w):
        def one(v, name):
            if norm == "layer":
                return torch.nn.functional.layer_norm(v, (cols,), w[name] + offset,
                                                      w[name + "_bias"], eps)
            return torch.nn.functional.rms_norm(v, (cols,), w[name] + offset, eps)
        n = one(x, "post") if "post" in w else x
        if "gate" in w:
            n = n * w["gate"].reshape(-1, cols).repeat_interleave(
                rows // (w["gate"].numel() // cols), 0)
        h = residual + scale * n
        return h, one(h, "pre") if "pre" in w else None

    h, y = forward(**t, **kw)
    got = ref.stream(**t, **args)
    torch.testing.assert_close(got[0], h, rtol=1e-12, atol=1e-12)
    stats = torch.cat((got[2], torch.tensor([[0.0, 1.0]], dtype=F64).expand(rows, 2)), -1)
    if y is not None:
        out = ref.after(h, **args)
        torch.testing.assert_close(out[0], y, rtol=1e-12, atol=1e-12)
        stats = torch.cat((got[2], out[2]), -1)
    g = torch.Generator().manual_seed(1)
    gh = torch.randn(rows, cols, generator=g, dtype=F64)
    gy = None if y is None else torch.randn(rows, cols, generator=g, dtype=F64)
    args.pop("eps")
    out = ref.block_norms_bwd(gh, gy, t["x"], h, stats, **args)
    names = ("x", "residual", "gate", "post", "post_bias", "pre", "pre_bias")
    leaves = {k: v.clone().requires_grad_() for k, v in {**t, **kw}.items()}

    def value(**w):
        h, y = forward(**w)
        return (h * gh).sum() + (0 if y is None else (y * gy).sum())

    value(**leaves).backward()
    for k, found in zip(names, out):
        if k not in leaves:
            assert found is None
            continue
        torch.testing.assert_close(found[0], leaves[k].grad, rtol=1e-11, atol=1e-11)
        step = 1e-5
        at = tuple(s // 2 for s in leaves[k].shape)
        moved = []
        for sign in (1, -1):
            other = {n: v.detach().clone() for n, v in leaves.items()}
            other[k][at] += sign * step
            moved.append(float(value(**other)))
        assert abs((moved[0] - moved[1]) / (2 * step) - float(found[0][at])) < 1e-7


def test_cross_entropy_reference(in_64_bits):
    g = torch.Generator().manual_seed(2)
    rows, width, vocab, scale = 7, 5, 11, 0.5
    h = torch.randn(rows, width, generator=g, dtype=F64, requires_grad=True)
    w = torch.randn(vocab, width, generator=g, dtype=F64, requires_grad=True)
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[2] = ref.IGNORE
    x = scale * h @ w.t()
    want = torch.nn.functional.cross_entropy(x, t, reduction="none")
    keep = (t != ref.IGNORE).double()
    (l, _), (lse, _) = ref.linear_cross_entropy(h.detach(), w.detach(), t, scale)
    torch.testing.assert_close(l, want.detach(), rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(lse, torch.logsumexp(x, -1).detach() * keep, rtol=1e-12, atol=1e-12)
    grads = torch.randn(2, rows, generator=g, dtype=F64)
    value = (want * grads[0] + torch.logsumexp(x, -1) * keep * grads[1]).sum()
    value.backward()
    (dh, _), (dw, _) = ref.linear_cross_entropy_bwd(grads[0], h.detach(), w.detach(), t, lse,
                                                    scale, grad_lse=grads[1])
    torch.testing.assert_close(dh, h.grad, rtol=1e-11, atol=1e-11)
    torch.testing.assert_close(dw, w.grad, rtol=1e-11, atol=1e-11)


# ---------------------------------------------------------------------------
# Products of fp32 values
# ---------------------------------------------------------------------------

def test_sizes_of_the_parts_tests_take_every_kernel(launches):
    calls = [(-1, op, *size, 4) for size in parts.SIZES
             for op in ("linear_cross_entropy", "linear_cross_entropy_bwd")]
    names = {name for made, _ in launches(*calls) for name, _, _ in made}
    names = subprocess.run(["c++filt"], input="\n".join(names), capture_output=True, check=True,
                           text=True).stdout.replace("hipo::(anonymous namespace)::", "")
    for tile in (128, 256):
        for epilogue in range(4):
            assert f"gemm<float, {tile}, (Epilogue){epilogue}, 3>" in names
    for n in (1, 2, 4):
        assert f"thin_hidden<float, {n}>" in names
        for grad in ("false", "true"):
            for groups in ((1,) if n == 4 else (1, 2)):
                assert f"thin_logits<float, {n}, {grad}, {groups}, false>" in names
    assert "thin_weight<float>" in names


def off_by(got, a, b):
    """The share of the products that are off by more than the bound."""
    want = a.double() * b.double()
    return float(((got - want).abs() > parts.TOL * want.abs()).double().mean())


@pytest.mark.parametrize("without", parts.PASSES)
def test_a_product_that_is_left_out_shows(without):
    """Of the operands that the kernels are tested with: with all six passes every
    product is within the bound, with five most are not."""
    for size in parts.SIZES[:8]:
        _, _, _, (h, w) = parts.one_logit_a_row(*size, "cpu")
        grad, hidden, weight, tokens, _ = parts.one_value_of_d_a_row(*size, "cpu")
        for a, b in ((w, h), (weight[tokens], -grad[:, None]), (hidden, -grad[:, None])):
            assert off_by(parts.product(a, b), a, b) == 0
            least = 0.5 if a.numel() > 100 else 0.3
            assert off_by(parts.product(a, b, without), a, b) > least, (size, without)


@pytest.mark.parametrize("without", parts.PASSES)
def test_a_logit_without_a_product_shows_in_its_probability(without):
    """e^(s - lse) where lse is s rounded, as the gradient's logits are tested."""
    for size in parts.SIZES:
        _, _, _, (h, w) = parts.one_logit_a_row(*size, "cpu")
        s = h.double() * w.double()
        lse = s.float().double()
        full, less = (torch.exp(parts.product(w, h, k) - lse) for k in (None, without))
        p = torch.exp(s - lse)
        tol = p * torch.expm1(parts.TOL * s.abs() + 2.0 ** -20)
        assert ((full - p).abs() <= tol).all()
        assert float(((less - p).abs() > tol).double().mean()) > 0.5 or size[0] < 10


@pytest.mark.parametrize("size", parts.SIZES[:8])
def test_operands_of_the_parts_tests(size):
    """They are what they say, by the 64-bit formulas."""
    hidden, weight, tokens, (h, w) = parts.one_logit_a_row(*size, "cpu")
    logits = hidden.double() @ weight.double().t()
    s = h.double() * w.double()
    rows = torch.arange(len(s))
    assert torch.equal(logits[rows, tokens], s)
    assert torch.equal(torch.logsumexp(logits, -1), s)
    grad, hidden, weight, tokens, lse = parts.one_value_of_d_a_row(*size, "cpu")
    (dh, _), (dw, _) = ref.linear_cross_entropy_bwd(grad, hidden, weight, tokens, lse)
    assert torch.equal(dh, -grad.double()[:, None] * weight.double()[tokens])
    want = torch.zeros_like(dw)
    want[tokens] = -grad.double()[:, None] * hidden.double()
    assert torch.equal(dw, want)
