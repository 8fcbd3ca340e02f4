"""The two ends of a language model, as its code calls them: how tokens enter
(the embedding lookup and its gradient) and how they leave (log probabilities
of given tokens, with entropy and top alternatives, and their gradient).

Each case is one call.  Where `own` is false, run() computes it with
elementary torch operations in fp32; where it is true, run() calls the
library's functions of the same meaning.
"""
import math
import os
import sys

import torch

own = False

BF16, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
_DTYPES = {"bf16": BF16, "f32": F32}
_BYTES = {"bf16": 2, "f32": 4}
IGNORE = -100


def _library():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "better-benchmark_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import hip_oracles
    return hip_oracles


def _logprobs(name, rows, vocab, dtype, **options):
    c = {"name": name, "op": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype,
         "scale": 1.0, "ignored": 0.0, "masked": False, "entropy": False, "top": 0}
    return {**c, **options}


def _logprobs_bwd(name, rows, vocab, dtype, **options):
    c = {"name": name, "op": "logprobs_bwd", "rows": rows, "vocab": vocab, "dtype": dtype,
         "scale": 1.0, "ignored": 0.0, "masked": False, "entropy": False, "lse": False}
    return {**c, **options}


def _embedding(name, tokens, width, vocab, dtype, **options):
    c = {"name": name, "op": "embedding", "tokens": tokens, "width": width, "vocab": vocab,
         "dtype": dtype, "scale": 1.0, "wide_ids": True}
    return {**c, **options}


def _embedding_bwd(name, tokens, width, vocab, dtype, **options):
    c = {"name": name, "op": "embedding_bwd", "tokens": tokens, "width": width, "vocab": vocab,
         "dtype": dtype, "out": dtype, "into": False, "scale": 1.0, "padding": 0.0,
         "wide_ids": True}
    return {**c, **options}


def listed():
    return [
        # One sequence's next token while it is generated: what the launch costs.
        _logprobs("logprobs_1x32000_top5", 1, 32000, "bf16", entropy=True, top=5),
        # A serving batch that returns the alternatives of every token.
        _logprobs("logprobs_64x128000_top20", 64, 128000, "bf16", scale=0.7, entropy=True,
                  top=20),
        # Scoring given texts with fp32 logits; an odd vocabulary, rows off 16 bytes.
        _logprobs("logprobs_1501x50001_f32", 1501, 50001, "f32", entropy=True),
        # A training step's loss: 4 sequences of 2048 tokens, prompts left out.
        _logprobs("logprobs_8192x128000", 8192, 128000, "bf16", ignored=0.125),
        # Policy gradient with an entropy bonus and a penalty on the normaliser.
        _logprobs_bwd("logprobs_bwd_1501x50001_f32", 1501, 50001, "f32", entropy=True, lse=True),
        # The same training step's gradient (the largest).
        _logprobs_bwd("logprobs_bwd_8192x128000", 8192, 128000, "bf16", ignored=0.125),
        # A decode step's lookup: launch and latency.
        _embedding("embedding_16x2048", 16, 2048, 32000, "bf16"),
        # The training step's lookup, scaled by sqrt(width).
        _embedding("embedding_8192x4096", 8192, 4096, 128000, "bf16", scale=64.0),
        # fp32 rows of an odd width, 32-bit ids.
        _embedding("embedding_20011x1001_f32", 20011, 1001, 50001, "f32", scale=0.5,
                   wide_ids=False),
        # A small model's embedding gradient.
        _embedding_bwd("embedding_bwd_2048x768", 2048, 768, 32000, "bf16"),
        # The training step's dense gradient.
        _embedding_bwd("embedding_bwd_8192x4096", 8192, 4096, 128000, "bf16", scale=64.0),
        # Gradient accumulation into an fp32 buffer (tied weights), padded batch.
        _embedding_bwd("embedding_bwd_16381x2880_into", 16381, 2880, 50001, "bf16", out="f32",
                       into=True, padding=0.125, wide_ids=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """A vocabulary or a width: half multiples of 64, a quarter of 8, the others any."""
    v = _log(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return max(step, v // step * step)


def draw(rng):
    op = rng.choice(("logprobs", "logprobs", "logprobs_bwd", "embedding", "embedding_bwd"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    vocab = _size(rng, 1000, 200000)
    if op in ("logprobs", "logprobs_bwd"):
        most = 8192 * 128000 * 2 // _BYTES[dtype] // vocab
        rows = _log(rng, 1, min(16384, most))
        c = {"op": op, "rows": rows, "vocab": vocab, "dtype": dtype,
             "scale": rng.choice((1.0, 1.0, 0.7, 1.25)),
             "ignored": rng.choice((0.0, 0.0, 0.25)), "masked": rng.random() < 0.25,
             "entropy": rng.random() < 0.5}
        if op == "logprobs_bwd":
            c["lse"] = rng.random() < 0.5
        else:
            c["top"] = rng.choice((0, 0, 1, 5, 20, 32)) if rows <= 512 else 0
        return c
    width = _size(rng, 64, 8192)
    vocab = min(vocab, (1 << 29) // width)
    tokens = _log(rng, 1, min(65536, (1 << 27) // width))
    c = {"op": op, "tokens": tokens, "width": width, "vocab": vocab, "dtype": dtype,
         "scale": rng.choice((1.0, 1.0, math.sqrt(width))), "wide_ids": rng.random() < 0.5}
    if op == "embedding_bwd":
        c["out"] = rng.choice((dtype, "f32"))
        c["into"] = rng.random() < 0.4
        c["padding"] = rng.choice((0.0, 0.0, 0.25))
    return c


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _token_ids(gen, count, vocab, device):
    """Token ids with the frequencies of text: the id's logarithm is uniform."""
    u = torch.rand(count, generator=gen, device=device, dtype=F64)
    ids = torch.floor(torch.exp(u * math.log(vocab + 1.0))) - 1.0
    return ids.clamp_(0, vocab - 1).to(I64)


def _left_out(gen, count, share, device):
    """Which of `count` places are left out: exactly int(count * share) of them."""
    out = torch.zeros(count, dtype=torch.bool, device=device)
    out[torch.randperm(count, generator=gen, device=device)[:int(count * share)]] = True
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    state = dict(case)
    vocab = case["vocab"]
    if case["op"] in ("logprobs", "logprobs_bwd"):
        rows = case["rows"]
        # Logits of a trained model: a wide body and a few tokens far above it.
        x = torch.randn(rows, vocab, generator=gen, device=dev, dtype=dt)
        x.mul_(2.5)
        peaks = torch.randint(0, vocab, (rows, 8), generator=gen, device=dev)
        x.scatter_(1, peaks, (8 + 6 * torch.rand(rows, 8, generator=gen, device=dev)).to(dt))
        tok = torch.where(torch.rand(rows, generator=gen, device=dev) < 0.7, peaks[:, 0],
                          _token_ids(gen, rows, vocab, dev))
        if case["masked"]:
            # Constrained decoding: one mask of the vocabulary, one token in ten
            # left, among them every token that is asked for.
            off = torch.rand(vocab, generator=gen, device=dev) < 0.9
            off[tok] = False
            x.masked_fill_(off, float("-inf"))
        tok[_left_out(gen, rows, case["ignored"], dev)] = IGNORE
        state.update(logits=x, ids=tok)
        if case["op"] == "logprobs_bwd":
            # The forward's results and the loss's gradients are in hand.
            lse = torch.empty(rows, device=dev)
            ent = torch.empty(rows, device=dev)
            for r in range(0, rows, 1024):
                ls = torch.log_softmax(x[r:r + 1024].float() * case["scale"], -1)
                p = ls.exp()
                ent[r:r + 1024] = -(p * torch.where(p > 0, ls, 0.0)).sum(-1)
                lse[r:r + 1024] = torch.logsumexp(x[r:r + 1024].float() * case["scale"], -1)
            keep = tok != IGNORE
            state["lse_in"] = torch.where(keep, lse, 0.0)
            state["grad"] = torch.randn(rows, generator=gen, device=dev) / rows
            state["entropy_in"] = torch.where(keep, ent, 0.0) if case["entropy"] else None
            state["grad_entropy"] = (0.1 * torch.randn(rows, generator=gen, device=dev) / rows
                                     if case["entropy"] else None)
            state["grad_lse"] = (0.1 * torch.randn(rows, generator=gen, device=dev) / rows
                                 if case["lse"] else None)
        return state
    count, width = case["tokens"], case["width"]
    ids = _token_ids(gen, count, vocab, dev)
    if case["op"] == "embedding":
        state["weight"] = (torch.randn(vocab, width, generator=gen, device=dev, dtype=dt) * 0.02)
    else:
        state["grad"] = torch.randn(count, width, generator=gen, device=dev, dtype=dt)
        state["padding_idx"] = None
        if case["padding"]:
            state["padding_idx"] = 1
            ids[_left_out(gen, count, case["padding"], dev)] = 1
        if case["into"]:
            state["buffer"] = torch.randn(vocab, width, generator=gen, device=dev,
                                          dtype=_DTYPES[case["out"]])
    state["ids"] = ids if case["wide_ids"] else ids.to(I32)
    return state


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    ho = _library()
    if s["op"] == "logprobs":
        return ho.token_logprobs(s["logits"], s["ids"], scale=s["scale"], ignore_index=IGNORE,
                                 entropy=s["entropy"], top=s["top"])
    if s["op"] == "logprobs_bwd":
        return ho.token_logprobs_bwd(s["grad"], s["logits"], s["ids"], s["lse_in"],
                                     scale=s["scale"], ignore_index=IGNORE,
                                     entropy=s["entropy_in"], grad_entropy=s["grad_entropy"],
                                     grad_lse=s["grad_lse"])
    if s["op"] == "embedding":
        return ho.embedding(s["weight"], s["ids"], scale=s["scale"])
    if s["into"]:
        return ho.embedding_bwd(s["grad"], s["ids"], s["vocab"], scale=s["scale"],
                                padding_idx=s["padding_idx"], into=s["buffer"])
    return ho.embedding_bwd(s["grad"], s["ids"], s["vocab"], scale=s["scale"],
                            padding_idx=s["padding_idx"], dtype=_DTYPES[s["out"]])


def _run_plain(s):
    return {"logprobs": _plain_logprobs, "logprobs_bwd": _plain_logprobs_bwd,
            "embedding": _plain_embedding, "embedding_bwd": _plain_embedding_bwd}[s["op"]](s)


def _order_key(x):
    """int64 keys of [R, V] values, the larger value first and, of equal ones,
    the lower index."""
    bits = (x.float() + 0.0).view(I32).to(I64)
    ordered = torch.where(bits < 0, -2147483648 - bits, bits)
    return ordered * (1 << 32) + torch.arange(x.shape[1] - 1, -1, -1, device=x.device)


def _plain_logprobs(s):
    keep = s["ids"] != IGNORE
    ids = torch.where(keep, s["ids"], 0)
    x = s["logits"].float() * s["scale"]
    t = x - x.amax(-1, keepdim=True)
    e = torch.exp(t)
    total = e.sum(-1)
    log_total = torch.log(total)
    lse = x.amax(-1) + log_total
    logprob = t.gather(1, ids[:, None])[:, 0] - log_total
    out = [torch.where(keep, logprob, 0.0), torch.where(keep, lse, 0.0)]
    if s["entropy"]:
        mean = torch.where(e > 0, e * t, 0.0).sum(-1) / total
        out.append(torch.where(keep, log_total - mean, 0.0))
    if s["top"]:
        which = torch.topk(_order_key(s["logits"]), s["top"], -1).indices
        value = t.gather(1, which) - log_total[:, None]
        out.append(torch.where(keep[:, None], value, float("-inf")))
        out.append(torch.where(keep[:, None], which, -1))
    return tuple(out)


def _plain_logprobs_bwd(s):
    keep = s["ids"] != IGNORE
    ids = torch.where(keep, s["ids"], 0)
    logp = s["logits"].float() * s["scale"] - s["lse_in"][:, None]
    p = torch.exp(logp)
    factor = -s["grad"]
    if s["lse"]:
        factor = factor + s["grad_lse"]
    g = p * factor[:, None]
    if s["entropy"]:
        part = s["grad_entropy"][:, None] * (logp + s["entropy_in"][:, None])
        g = g - torch.where(p > 0, p * part, 0.0)
    g.scatter_add_(1, ids[:, None], s["grad"][:, None])
    g = torch.where(keep[:, None], g * s["scale"], 0.0)
    return g.to(s["logits"].dtype)


def _plain_embedding(s):
    rows = s["weight"][s["ids"].long()].float()
    return (rows * s["scale"]).to(s["weight"].dtype)


def _plain_embedding_bwd(s):
    ids = s["ids"].long()
    grad = s["grad"].float()
    if s["padding_idx"] is not None:
        grad = torch.where((ids != s["padding_idx"])[:, None], grad, 0.0)
    total = torch.zeros(s["vocab"], s["width"], device=grad.device)
    total.index_add_(0, ids, grad)
    total = total * s["scale"]
    if s["into"]:
        return s["buffer"].copy_(s["buffer"].float() + total)
    return total.to(_DTYPES[s["out"]])


# ---------------------------------------------------------------------------
# What a pass cannot do without, and its exact result
# ---------------------------------------------------------------------------

def _distinct(case):
    """Expected number of distinct ids that are not left out."""
    v = torch.arange(1, case["vocab"] + 1, dtype=F64)
    p = torch.log((v + 1) / v) / math.log(case["vocab"] + 1.0)
    count = case["tokens"] - int(case["tokens"] * case.get("padding", 0.0))
    return float((1 - (1 - p) ** count).sum())


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] in ("logprobs", "logprobs_bwd"):
        rows = case["rows"]
        kept = rows - int(rows * case["ignored"])
        if case["op"] == "logprobs":
            outs = 8 + 4 * case["entropy"] + 12 * case["top"]
            return {"bytes": kept * case["vocab"] * e + rows * (8 + outs),
                    "flops": kept * case["vocab"] * (4 + 2 * case["entropy"])}
        ins = 16 + 8 * case["entropy"] + 4 * case["lse"]
        return {"bytes": (kept + rows) * case["vocab"] * e + rows * ins,
                "flops": kept * case["vocab"] * (4 + 3 * case["entropy"])}
    count, width = case["tokens"], case["width"]
    ids = count * (8 if case["wide_ids"] else 4)
    if case["op"] == "embedding":
        return {"bytes": (count + _distinct(case)) * width * e + ids, "flops": count * width}
    kept = count - int(count * case["padding"])
    out = _BYTES[case["out"]]
    written = 2 * _distinct(case) * out if case["into"] else case["vocab"] * out
    return {"bytes": kept * width * e + written * width + ids,
            "flops": kept * width + _distinct(case) * width}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "logprobs_bwd":
        return _exact_logprobs_bwd(s)
    ids = s["ids"].long()
    if case["op"] == "embedding":
        return torch.nn.functional.embedding(ids, s["weight"].double()) * case["scale"]
    # One product per block of columns with the matrix of (token, position).
    there = torch.ones_like(ids, dtype=F64)
    if s["padding_idx"] is not None:
        there[ids == s["padding_idx"]] = 0
    where = torch.stack((ids, torch.arange(ids.numel(), device=ids.device)))
    pick = torch.sparse_coo_tensor(where, there, (case["vocab"], ids.numel()))
    out = torch.empty(case["vocab"], case["width"], dtype=F64, device=ids.device)
    for c in range(0, case["width"], 512):
        out[:, c:c + 512] = torch.sparse.mm(pick, s["grad"][:, c:c + 512].double().contiguous())
    out *= case["scale"]
    return out + s["buffer"].double() if case["into"] else out


def _exact_logprobs(s):
    outs = [[], [], [], []]
    for r in range(0, s["rows"], 512):
        ids = s["ids"][r:r + 512]
        skip = ids == IGNORE
        ls = torch.log_softmax(s["logits"][r:r + 512].double() * s["scale"], -1)
        own_token = torch.nn.functional.one_hot(ids.clamp(min=0), s["vocab"]).bool()
        outs[0].append(ls[own_token].masked_fill(skip, 0))
        outs[1].append(torch.logsumexp(s["logits"][r:r + 512].double() * s["scale"], -1)
                       .masked_fill(skip, 0))
        if s["entropy"]:
            outs[2].append(torch.special.entr(ls.exp()).sum(-1).masked_fill(skip, 0))
        if s["top"]:
            best = ls.sort(-1, descending=True).values[:, :s["top"]]
            outs[3].append(best.masked_fill(skip[:, None], float("-inf")))
    result = [torch.cat(o) for o in outs if o]
    return tuple(result + ([None] if s["top"] else []))


def _exact_logprobs_bwd(s):
    out = torch.empty(s["rows"], s["vocab"], dtype=F64, device=s["logits"].device)
    for r in range(0, s["rows"], 512):
        rows = slice(r, r + 512)
        ids = s["ids"][rows]
        ls = s["logits"][rows].double() * s["scale"]
        ls = ls - s["lse_in"][rows, None].double()
        p = ls.exp()
        g = torch.nn.functional.one_hot(ids.clamp(min=0), s["vocab"]).double() - p
        g *= s["grad"][rows, None].double()
        if s["lse"]:
            g += s["grad_lse"][rows, None].double() * p
        if s["entropy"]:
            # -p (ln p + H), with entr(p) = -p ln p
            g += s["grad_entropy"][rows, None].double() * (
                torch.special.entr(p) - p * s["entropy_in"][rows, None].double())
        out[rows] = (g * s["scale"]).masked_fill((ids == IGNORE)[:, None], 0)
    return out
