"""tk_sample_tokens where the cut of top-p lies among weights far below the largest, whose number makes up the sum: the
oracle's sums have 64 bits of mantissa, and every row is asked.

What the kernel's f64 sums may be off by, as a share of all: a lane adds up vocab / (512 * CTAs) weights one after the
other and some 20 partial sums follow, half a step of f64 each; a weight itself is within 2e-14 of its value (a
polynomial's 9e-15, and 43 octaves of an exponent that is rounded to 2^-53); units of 2^-52 (a list) or 2^-45 of a
bin's largest weight.  The inputs keep the goal further from the ranks' borders than that (asserted before the call), so
counts and tokens have to be equal."""
from decimal import Decimal, getcontext
from fractions import Fraction

import numpy as np
import pytest

from test_kv4_gpu import kind
from tiny_kernel import ops

pytestmark = pytest.mark.gpu

getcontext().prec = 60


def off_by(vocab, ctas=1):
    return (vocab / (512 * ctas) + 20) * 2.0**-53


def sample(torch, dev, l, dtype, top_p, u, top_k=None, min_p=None):
    """(tokens, kept) of rows of logits."""
    rows, vocab = l.shape
    x = torch.from_numpy(np.ascontiguousarray(l, np.float32)).cuda().to(kind(torch, dtype))
    each = lambda v, t: None if v is None else torch.tensor(np.broadcast_to(v, (rows,)).copy(), dtype=t, device="cuda")
    tokens, kept = (torch.full((rows,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    ops.sample_tokens(dev, x, None, each(top_k, torch.int32), each(top_p, torch.float32), each(min_p, torch.float32),
                      each(u, torch.float32), tokens, kept, rows, vocab, dtype)
    return tokens.cpu().numpy(), kept.cpu().numpy()


TAILS = [
    # vocab, logit of all but one token, top_p
    (128256, -20.25, 0.9999), (128256, -22.5, 0.99999), (128256, -25.0, 0.999999), (128256, -27.0, 0.9999999),
    (393216, -29.25, 0.99999994), (50257, -18.0, 0.9995), (32000, -23.25, 0.9999995), (1500, -13.5, 0.999),
]


def tail(vocab, low, top_p):
    """How many tokens are kept, and how far (in tokens) the goal is from a border: one token of weight 1, the others of
    one weight w, in whole numbers and 60 digits."""
    w = Decimal(low).exp()
    p = Fraction(float(np.float32(top_p)))
    goal = Decimal(p.numerator) / Decimal(p.denominator) * (1 + (vocab - 1) * w)
    tokens = (goal - 1) / w
    whole = int(tokens)
    return 1 + whole + 1, float(min(tokens - whole, whole + 1 - tokens)), float(w)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 40, 80])
@pytest.mark.parametrize("vocab,low,top_p", TAILS)
def test_tails_of_one_weight(torch_cuda, tkdev, vocab, low, top_p, rows, dtype):
    """Of equal weights the first by index are kept."""
    at = np.arange(rows) * 37 % vocab
    l = np.full((rows, vocab), low)
    l[np.arange(rows), at] = 0.0
    for top_k in (None, vocab - 1):  # the latter leaves out the last of the tail
        want, margin, w = tail(vocab if top_k is None else top_k, low, top_p)
        assert margin > off_by(vocab, 4 if vocab > 300000 else 1) / w + vocab * 2.0**-44
        last = np.maximum(at, want - 1)  # of the kept ones, by index: the first of the tail, and the one above it
        for u, token in ((1.0, last), (0.0, np.zeros(rows)), (0.5, at)):
            tokens, kept = sample(torch_cuda, tkdev, l, dtype, top_p, u, top_k)
            assert (kept == want).all() and (tokens == token).all()


BOUND = off_by(128256) + 2e-14 + 2.0**-45


def ranked(l, top_p, u, bound):
    """(token, kept) of a row, in numbers of 64 bits of mantissa; the distances of both goals from the nearest border
    have to be above `bound` of the sums."""
    order = np.argsort(-l, kind="stable")
    x = l.astype(np.longdouble)
    w = np.exp(x - x[order[0]])
    passed = np.cumsum(w[order])
    goal = np.longdouble(top_p) * passed[-1]
    kept = 1 + int(np.searchsorted(passed, goal))
    assert np.abs(passed - goal).min() > bound * passed[-1]
    at = np.sort(order[:kept])
    passed = np.cumsum(w[at])
    goal = np.longdouble(u) * passed[-1]
    assert np.abs(passed - goal).min() > bound * passed[-1]
    return int(at[np.searchsorted(passed, goal, side="right")]), kept


SPREAD = [
    # vocab, middle of all but one token, width, top_p: a few hundred tokens of a bin (a list), thousands of different
    # ones (their digits), bins far apart
    (128256, -25.0, 2.0, 0.99999), (128256, -22.5, 0.001, 0.99999), (128256, -20.0, 0.05, 0.9999), (50257, -24.0, 0.3, 0.999999),
    (128256, -12.0, 1.0, 0.7), (60000, -16.0, 0.01, 0.996), (4000, -19.0, 0.5, 0.99999),
]


def spread(vocab, middle, width, rows):
    rng = np.random.default_rng(int(-middle * 100) + vocab + rows)
    l = (rng.normal(size=(rows, vocab)) * width + middle).astype(np.float32)
    l[np.arange(rows), rng.integers(0, vocab, rows)] = 0.0
    return l, rng.uniform(0.9999, 1, rows).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 30])
@pytest.mark.parametrize("vocab,middle,width,top_p", SPREAD)
def test_tails_of_many_weights(torch_cuda, tkdev, vocab, middle, width, top_p, rows, dtype):
    torch = torch_cuda
    l, u = spread(vocab, middle, width, rows)
    l = torch.from_numpy(l).to(kind(torch, dtype)).float().numpy()
    want = [ranked(row, np.float32(top_p), u[i], BOUND) for i, row in enumerate(l)]
    tokens, kept = sample(torch, tkdev, l, dtype, top_p, u)
    assert list(zip(tokens.tolist(), kept.tolist())) == want
