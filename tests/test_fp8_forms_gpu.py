"""GPU parity of tk_fp8_matmul in each form and way over its tiles (the shapes of test_fp8_forms_cpu.py, which asserts what
each takes), against the f64 oracle.  Whole numbers below 2^24 are exact in f32, and round once to a 16-bit type; for others
the bounds are those of test_fp8_gpu.py."""
import functools

import numpy as np
import pytest

from test_fp8_forms_cpu import FORMS
from test_fp8_gpu import operands, product
from test_kv4_gpu import HALF_STEP, LEAST, f64, kind
from tiny_kernel import ops

pytestmark = pytest.mark.gpu

SHAPES = sorted(FORMS)
named = pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))


@functools.lru_cache(maxsize=1)
def whole(torch, shape):
    return operands(torch, sum(shape), *shape, whole=True, pad=shape[0] % 2)


@named
@pytest.mark.parametrize("dtype,gap,offset", [("f32", 0, 0), ("f32", 3, 1), ("f16", 1, 1), ("bf16", 0, 0), ("bf16", 16, 0)])
def test_whole_numbers_are_exact(torch_cuda, tkdev, shape, dtype, gap, offset):
    """Rows of the output on their 32-byte boundary and off it."""
    t, want, size = whole(torch_cuda, shape)
    assert size.max() < 2**24
    got = product(torch_cuda, tkdev, t, *shape, dtype, gap=gap, offset=offset)
    rounded = torch_cuda.from_numpy(want).float().to(kind(torch_cuda, dtype))
    assert torch_cuda.equal(got.cpu(), rounded)


@named
def test_any_numbers(torch_cuda, tkdev, shape):
    m, k, n = shape
    t, want, size = operands(torch_cuda, 3 * m + k + n, m, k, n, whole=False)
    error = (128 + 3 + -(-k // 128)) * 2.0**-23
    for dtype in ("f32", "bf16"):
        got = f64(product(torch_cuda, tkdev, t, m, k, n, dtype))
        assert (np.abs(got - want) <= error * size + HALF_STEP[dtype] * np.abs(want) + LEAST[dtype]).all()
        if dtype == "f32":
            assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


@named
def test_nan_stays_in_its_rows_and_columns(torch_cuda, tkdev, shape):
    """A code of a's last row, a scale of its first, a code of w's last row; the last block of k."""
    torch, (m, k, n) = torch_cuda, shape
    t, want, _ = operands(torch, 7, m, k, n, whole=True)
    t[2][n - 1, k - 1] = 0xFF
    bad_rows = [m - 1] if m > 1 else []
    for r in bad_rows:
        t[0][r, k - 1] = 0x7F
    if m > 2:
        t[1][0, 0] = float("nan")
        bad_rows.append(0)
    got = f64(product(torch, tkdev, t, m, k, n, "f32"))
    bad = np.zeros((m, n), bool)
    bad[bad_rows] = bad[:, n - 1] = True
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])


@named
def test_scales_as_far_as_their_product_fits(torch_cuda, tkdev, shape):
    """Blocks whose scales multiply to 2^127, 2^-126 and, below that, a multiple of 2^-149, over sums of 0, 1 and -1: exact."""
    torch, (m, k, n) = torch_cuda, shape
    stride, blocks = -(-k // 16) * 16, -(-k // 128)
    for a_scale, w_scale in ((2.0**100, 2.0**27), (2.0**-120, 2.0**-6), (2.0**-126, 2.0**-20), (1.0, 2.0**127)):
        a, w = (torch.zeros((r, stride), dtype=torch.uint8, device="cuda") for r in (m, n))
        a[:, 0] = 0x38                         # 1 in the first place of every row,
        w[::3, 0], w[1::3, 0] = 0x38, 0xB8     # 1, -1 and 0 in that of the columns
        scales = [torch.full((r, blocks), s, device="cuda") for r, s in ((m, a_scale), (-(-n // 128), w_scale))]
        got = product(torch, tkdev, [a, scales[0], w, scales[1]], m, k, n, "f32")
        want = torch.zeros(n, device="cuda")
        want[::3], want[1::3] = a_scale * w_scale, -a_scale * w_scale
        assert torch.equal(got, want.expand(m, n))


@named
def test_the_same_bits_whenever_it_runs(torch_cuda, tkdev, shape):
    """Again, on two streams at once with another product's operands, and captured and replayed over other operands."""
    torch, (m, k, n) = torch_cuda, shape
    a, b = (operands(torch, seed, m, k, n, whole=False)[0] for seed in (1, 2))
    want = [product(torch, tkdev, t, m, k, n, "bf16").clone() for t in (a, b)]
    outs = [torch.zeros((m, n), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    stride = a[0].shape[1]
    torch.cuda.synchronize()

    def call(t, out, stream):
        ops.fp8_matmul(tkdev, *t, out, m, k, n, "bf16", a_stride=stride, w_stride=stride, stream=stream.cuda_stream, sync=False)

    for _ in range(5):
        for t, out, s in zip((a, b), outs, streams):
            call(t, out, s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        call(a, outs[0], streams[0])
    for other in (b, a):
        keep = [v.clone() for v in a]
        for to, v in zip(a, other):
            to.copy_(v)
        outs[0].zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[1] if other is b else want[0])
        for to, v in zip(a, keep):
            to.copy_(v)
    del graph
