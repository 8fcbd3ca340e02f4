"""Products of fp32 values as the matrix cores take them: three bf16 parts of
each value, six products of parts.  Operands of the output layer of which every
result is one such product, so that a part, a product of parts or a plane that is
missing shows in each of them."""
import torch

F32, F64 = torch.float32, torch.float64

PASSES = [(0, 2), (2, 0), (1, 1), (1, 0), (0, 1), (0, 0)]

# What one product may be off by, relative to itself: a step, 2^-23, for the last
# addition (a matrix instruction may cut its sums), 2^-7 of it for the five before,
# whose sums are below 2^-7 of the product, and the three products of parts that
# are left out, below 3 * 2^-26.  The parts hold all 24 bits.
TOL = 2.0 ** -22

SELECTORS = 8


def split(x):
    """Three bf16 parts of fp32 values, in 64 bits."""
    parts, rest = [], x.float()
    for _ in range(3):
        p = rest.to(torch.bfloat16).float()
        parts.append(p.double())
        rest = rest - p
    return parts


def product(a, b, without=None):
    """a b as the passes give it, one left out."""
    pa, pb = split(a), split(b)
    return sum(pa[i] * pb[j] for i, j in PASSES if (i, j) != without)


def one_logit_a_row(rows, width, vocab, device, seed=0):
    """(hidden, weight, tokens, s): a row's logit of its token is s = one value of
    hidden times one of the weight, the others are 1e5 below.  The tokens are 8 of
    the vocabulary, from its first to its last; hidden's value is in another column
    from row to row, beside a 1 in one of the last 8, in which the weight is 0 for
    the row's token and -1e5 for the others."""
    g = torch.Generator(device=device).manual_seed(seed)
    free = width - SELECTORS
    at = torch.linspace(0, vocab - 1, SELECTORS, device=device).round().long()
    weight = torch.randn(vocab, width, generator=g, device=device) * 30
    weight[:, free:] = -1e5
    weight[at, torch.arange(free, width, device=device)] = 0.0
    row = torch.arange(rows, device=device)
    k, c = row * 37 % free, row % SELECTORS
    value = torch.randn(rows, generator=g, device=device) * 30
    hidden = torch.zeros(rows, width, device=device)
    hidden[row, k] = value
    hidden[row, free + c] = 1.0
    tokens = at[c]
    return hidden, weight, tokens, (value, weight[tokens, k])


def one_value_of_d_a_row(rows, width, vocab, device, seed=0):
    """(grad, hidden, weight, tokens, lse): every probability is 0, so that d is
    -grad at the token and 0 elsewhere; no token is in two rows.  dhidden is
    -grad weight[token], dweight[token] is -grad hidden, and 0 elsewhere."""
    g = torch.Generator(device=device).manual_seed(seed)
    hidden = torch.randn(rows, width, generator=g, device=device)
    weight = torch.randn(vocab, width, generator=g, device=device)
    tokens = torch.randperm(vocab, generator=g, device=device)[:rows]
    grad = torch.randn(rows, generator=g, device=device)
    return grad, hidden, weight, tokens, torch.full((rows,), 1e9, device=device)


# (rows, width, vocabulary) by which fp32 operands take every kernel that
# multiplies: those of up to 16, 32 and 64 rows, K split among groups of waves or
# not, the products of small and of large tiles, for the logits and both gradients.
SIZES = [(3, 65, 700), (20, 100, 900), (50, 100, 900), (3, 65, 20001), (20, 100, 20001),
         (50, 100, 20001), (100, 72, 300), (300, 100, 1500), (2100, 100, 33000),
         (2100, 1000, 9000)]
