"""tk_sample_tokens where a row's CTAs have slices of a few tokens, or of none: small vocabularies with top-p alone, in
rows that are flat, whose list of the largest is not likely to hold the sum, and rows that are not.  All CTAs of a row have
to take the same way.  Every row is asked: the inputs keep away from the borders of the oracle's comparisons."""
import numpy as np
import pytest

import fp8
from test_kv4_gpu import kind
from tiny_kernel import ops

pytestmark = pytest.mark.gpu

VOCABS = [1, 3, 9, 17, 23, 60, 100, 103, 130, 150, 200, 257, 258, 259, 390, 450, 451, 455, 500]


def inputs(vocab, rows):
    """Rows of normal logits of three widths, some of them with equal values, and their parameters."""
    rng = np.random.default_rng(vocab * 1000 + rows)
    l = rng.normal(size=(rows, vocab)) * np.array([0.5, 1.0, 2.0])[np.arange(rows) % 3][:, None]
    l[3::7] = np.round(l[3::7] * 4) / 4
    top_k = np.array([0, -1, vocab, vocab + 5])[np.arange(rows) % 4].astype(np.int32)
    return l.astype(np.float32), rng.uniform(0.05, 0.99, rows).astype(np.float32), top_k, rng.random(rows).astype(np.float32)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 2, 37, 38, 74, 75, 148, 149])
@pytest.mark.parametrize("vocab", VOCABS)
def test_slices_of_few_tokens(torch_cuda, tkdev, vocab, rows, dtype):
    """Eight, four, two and one CTA a row, as top-p alone or with an array of top-k that asks for none has them."""
    torch = torch_cuda
    l, top_p, top_k, u = inputs(vocab, rows)
    x = torch.from_numpy(l).cuda().to(kind(torch, dtype))
    p, k, r = (torch.from_numpy(v).cuda() for v in (top_p, top_k, u))
    want = []
    for i, row in enumerate(x.double().cpu().numpy()):
        token, kept, slack = fp8.sample(row, None, None, top_p[i], None, u[i])
        assert slack > 1e-9
        want.append((token, kept))
    for filters in (None, k):
        tokens, kept = (torch.full((rows,), -7, dtype=torch.int32, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        # rows of a stride that keeps each on its 16-byte boundary: of any stride, only some are
        for stride in (vocab, -(-vocab // 8) * 8):
            held = torch.full((rows, stride), 99.0, dtype=x.dtype, device="cuda")
            held[:, :vocab] = x
            torch.cuda.synchronize()
            ops.sample_tokens(tkdev, held, None, filters, p, None, r, tokens, kept, rows, vocab, dtype, stride=stride)
            assert list(zip(tokens.tolist(), kept.tolist())) == want
