"""GPU parity of the 8-bit projections (tk_add_rmsnorm_fp8, tk_fp8_quantize, tk_fp8_matmul) against the f64
oracle.

Norm: s rounds once (2 of it enter), its squares' sum at most 32 + 5 + 32 + 1 times, which the root halves, mean,
root (2 steps) and two products follow, and the scale's division: less than 48 * 2^-24 in all.  A code is within half
a step of what it stands for: 2^-4 of it, or 2^-10 where it is below 2^-6.  The sum is rounded twice, to f32 and to
its type.
Product: whole numbers below 2^24 are exact.  Otherwise sums of f32 that round either way (2^-23 a product or
scale, at most 128 + 3 in a block, one for each block after it) and half a step of the output's type; what the tensor
cores do is well inside that, so the 2-norm of f32 outputs is held to 1e-6 of it as well, as for f32 operations.
"""
import numpy as np
import pytest

import fp8
from test_kv4_gpu import HALF_STEP, LEAST, f64, kind
from tiny_kernel import ops

pytestmark = pytest.mark.gpu

NORM_ERROR = 48 * 2.0**-24


def rows_of(torch, seed, rows, dim, dtype, gap, offset=0):
    """Rows of channels of different size, gap elements apart, offset elements off their allocation's start."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    held = torch.full((offset + rows * (dim + gap),), 7.0, dtype=kind(torch, dtype), device="cuda")
    x = held[offset:].view(rows, dim + gap)[:, :dim]
    size = torch.exp(torch.randn(dim, generator=g, device="cuda"))
    x.copy_(torch.randn((rows, dim), generator=g, device="cuda") * size)
    return x


def codes_of(torch, rows, dim, gap, offset=0):
    held = torch.full((offset + rows * (dim + gap),), 0x55, dtype=torch.uint8, device="cuda")
    return held, held[offset:].view(rows, dim + gap)


def check_codes(y, codes, scales, want_scales, block_rows, error):
    """Codes and scales of y (f64), whose values may be off by `error` of theirs."""
    rows, dim = y.shape
    assert scales.shape == want_scales.shape
    nan = np.isnan(want_scales)
    assert np.array_equal(np.isnan(scales), nan)
    assert (np.abs(scales - want_scales)[~nan] <= (error + 2.0**-23) * want_scales[~nan]).all()
    each = fp8.spread(scales, rows, dim, block_rows)
    fine = ~np.isnan(each)
    assert (codes[~fine] == 0).all()
    v, back = np.abs(y[fine]) / each[fine], fp8.TABLE[codes[fine]] * each[fine]
    off = np.abs(back - y[fine]) / each[fine]
    bound = np.maximum(v * 2.0**-4, 2.0**-10) + (error + 3 * 2.0**-24) * v
    assert (off <= bound).all(), (off - bound).max()


NORMS = [
    # rows, dim, residual, weight, gap, offset
    (1, 4096, True, True, 0, 0), (5, 4096, False, True, 0, 0), (3, 1, True, True, 0, 0), (2, 7, True, False, 3, 1),
    (9, 128, True, True, 0, 0), (4, 129, False, False, 0, 0), (33, 200, True, True, 8, 0), (2, 32768, True, True, 0, 0),
    (7, 14336, True, True, 16, 0), (400, 640, True, True, 0, 0), (301, 1000, True, True, 1, 1), (297, 256, False, True, 0, 0),
    (310, 5120, True, True, 0, 4), (299, 16384, True, True, 0, 0), (300, 1032, True, False, 0, 0), (1000, 72, True, True, 0, 0),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", NORMS, ids=lambda c: "-".join(map(str, c)))
def test_norm(torch_cuda, tkdev, case, dtype):
    torch = torch_cuda
    rows, dim, has_residual, has_weight, gap, offset = case
    x = rows_of(torch, dim, rows, dim, dtype, gap, offset)
    r = rows_of(torch, dim + 1, rows, dim, dtype, 2 * gap, offset) if has_residual else None
    w = torch.randn(dim, device="cuda") if has_weight else None
    total = torch.full((rows, dim + gap), 9.0, dtype=kind(torch, dtype), device="cuda")
    held, codes = codes_of(torch, rows, dim, gap, offset)
    scales = torch.full((rows, -(-dim // 128)), -1.0, device="cuda")
    want_sum, y = fp8.add_rmsnorm(f64(x), f64(r) if has_residual else None, f64(w) if has_weight else None, 1e-5)
    torch.cuda.synchronize()
    ops.add_rmsnorm_fp8(tkdev, x, r, w, total, codes, scales, rows, dim, 1e-5, dtype, x_stride=dim + gap,
                        residual_stride=dim + 2 * gap, sum_stride=dim + gap, codes_stride=dim + gap)
    check_codes(y, codes[:, :dim].cpu().numpy(), f64(scales), fp8.group_scales(y, 1), 1, NORM_ERROR)
    got = f64(total)
    assert (np.abs(got[:, :dim] - want_sum) <= (HALF_STEP[dtype] + 2.0**-24) * np.abs(want_sum) + LEAST[dtype]).all()
    assert (got[:, dim:] == 9).all() and (codes[:, dim:] == 0x55).all() and (held[:offset] == 0x55).all()


@pytest.mark.parametrize("place", ["x", "residual"])
def test_norm_in_place(torch_cuda, tkdev, place):
    torch = torch_cuda
    x, r = (rows_of(torch, s, 40, 1536, "bf16", 0) for s in (1, 2))
    w = torch.ones(1536, device="cuda")
    out = []
    for inplace in (False, True):
        a, b = x.clone(), r.clone()
        total = (a if place == "x" else b) if inplace else torch.empty_like(x)
        codes, scales = torch.empty((40, 1536), dtype=torch.uint8, device="cuda"), torch.empty((40, 12), device="cuda")
        torch.cuda.synchronize()
        ops.add_rmsnorm_fp8(tkdev, a, b, w, total, codes, scales, 40, 1536, 1e-6, "bf16")
        out.append((total, codes, scales))
    assert all(torch.equal(p, q) for p, q in zip(*out))


def test_norm_of_zeros_and_what_is_not_finite(torch_cuda, tkdev):
    torch = torch_cuda
    x = rows_of(torch, 3, 6, 512, "f32", 0)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 200] = float("inf")
    x[3, 128:256] = 0
    codes, scales = torch.full((6, 512), 1, dtype=torch.uint8, device="cuda"), torch.zeros((6, 4), device="cuda")
    torch.cuda.synchronize()
    ops.add_rmsnorm_fp8(tkdev, x, None, None, None, codes, scales, 6, 512, 1e-5)
    c, s = codes.cpu().numpy(), scales.cpu().numpy()
    assert (c[0] == 0).all() and (s[0] == 2.0**-126).all()
    assert np.isnan(s[1]).all() and (c[1] == 0).all()        # the root of NaN reaches the whole row
    assert np.isnan(s[2, 1]) and (s[2, [0, 2, 3]] == 2.0**-126).all() and (c[2] & 127 == 0).all()  # 1 / inf is 0
    assert s[3, 1] == np.float32(2.0**-126) and (c[3, 128:256] == 0).all() and np.isfinite(s[3]).all()


QUANTIZED = [(1, 1), (1, 128), (3, 129), (16, 96), (127, 300), (128, 128), (129, 256), (300, 1000), (64, 14336), (1000, 40)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [1, 128])
@pytest.mark.parametrize("rows,dim", QUANTIZED)
@pytest.mark.parametrize("gap,offset", [(0, 0), (8, 0), (3, 1)])
def test_quantize(torch_cuda, tkdev, rows, dim, block, dtype, gap, offset):
    torch = torch_cuda
    x = rows_of(torch, rows + dim, rows, dim, dtype, gap, offset)
    if rows > 2 and dim > 128:  # groups of nothing, of one size, and of what is not finite
        x[0, :128] = 0
        x[1, 3], x[2, 128] = float("inf"), float("nan")
    held, codes = codes_of(torch, rows, dim, gap, offset)
    scales = torch.full((-(-rows // block), -(-dim // 128)), -1.0, device="cuda")
    torch.cuda.synchronize()
    ops.fp8_quantize(tkdev, x, codes, scales, rows, dim, block, dtype, x_stride=dim + gap, codes_stride=dim + gap)
    y = f64(x)
    check_codes(np.where(np.isfinite(y), y, 0), codes[:, :dim].cpu().numpy(), f64(scales), fp8.group_scales(y, block), block, 0)
    assert (codes[:, dim:] == 0x55).all() and (held[:offset] == 0x55).all()


def test_quantize_keeps_small_and_large_values(torch_cuda, tkdev):
    """Groups of subnormals, of the largest f32 values, and of one size."""
    torch = torch_cuda
    x = torch.zeros((4, 128), device="cuda")
    x[0] = torch.linspace(-1e-38, 1e-38, 128, device="cuda")
    x[1] = torch.linspace(-3.4e38, 3.4e38, 128, device="cuda")
    x[2] = -0.3
    codes, scales = torch.zeros((4, 128), dtype=torch.uint8, device="cuda"), torch.zeros((4, 1), device="cuda")
    torch.cuda.synchronize()
    ops.fp8_quantize(tkdev, x, codes, scales, 4, 128)
    y = f64(x)
    check_codes(y, codes.cpu().numpy(), f64(scales), fp8.group_scales(y, 1), 1, 0)
    assert (codes[2] == 0xFE).all()  # -448


# ---- the product -----------------------------------------------------------------------------------

def operands(torch, seed, m, k, n, whole, pad=0):
    """Codes (rows on 16-byte boundaries, what lies past k is anything) and scales; whole: small whole numbers and
    powers of two, whose sums are exact."""
    rng = np.random.default_rng(seed)
    stride = -(-k // 16) * 16 + 16 * pad
    blocks = -(-k // 128)
    if whole:
        of = {v: c for c, v in enumerate(fp8.TABLE[:128])}
        small = np.array([of[float(abs(v))] | (0x80 if v < 0 else 0) for v in range(-4, 5)], np.uint8)
        a, w = (small[rng.integers(0, 9, (r, stride))] for r in (m, n))
        a_scales, w_scales = (2.0 ** rng.integers(0, 3, (r, blocks)) for r in (m, -(-n // 128)))
    else:
        a, w = (rng.integers(0, 255, (r, stride)).astype(np.uint8) for r in (m, n))
        a, w = (np.where((c & 127) == 127, 0, c).astype(np.uint8) for c in (a, w))
        a_scales, w_scales = (np.exp(rng.normal(size=(r, blocks))) * 1e-2 for r in (m, -(-n // 128)))
    a_scales, w_scales = a_scales.astype(np.float32), w_scales.astype(np.float32)
    t = [torch.from_numpy(v).cuda() for v in (a, a_scales, w, w_scales)]
    want, size = fp8.matmul(a[:, :k], a_scales, w[:, :k], w_scales)
    return t, want, size


def product(torch, dev, t, m, k, n, dtype, gap=0, offset=0, **more):
    held = torch.full((offset + m * (n + gap),), 7.0, dtype=kind(torch, dtype), device="cuda")
    out = held[offset:].view(m, n + gap)
    torch.cuda.synchronize()
    ops.fp8_matmul(dev, *t, out, m, k, n, dtype, a_stride=t[0].shape[1], w_stride=t[2].shape[1], out_stride=n + gap, **more)
    torch.cuda.synchronize()
    assert (held[:offset] == 7).all() and (out[:, n:] == 7).all()
    return out[:, :n]


SHAPES = [
    # m, k, n
    (1, 1, 1), (1, 128, 128), (1, 16, 3), (2, 127, 129), (5, 129, 127), (15, 1000, 64), (16, 640, 256), (17, 300, 200),
    (31, 2048, 130), (33, 384, 1000), (64, 1536, 257), (65, 2000, 333), (100, 4096, 640), (127, 96, 140), (128, 512, 128),
    (129, 1100, 129), (200, 257, 500), (255, 768, 255), (256, 512, 512), (300, 1024, 1300), (513, 900, 777),
    (700, 2048, 300), (1030, 640, 1100),
]


@pytest.mark.parametrize("m,k,n", SHAPES)
def test_product_of_whole_numbers_is_exact(torch_cuda, tkdev, m, k, n):
    t, want, size = operands(torch_cuda, m + k + n, m, k, n, whole=True, pad=m % 2)
    assert size.max() < 2**24
    assert np.array_equal(f64(product(torch_cuda, tkdev, t, m, k, n, "f32", gap=n % 3, offset=m % 2)), want)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m,k,n", [s for s in SHAPES if s[0] * s[1] * s[2] > 1e5])
def test_product(torch_cuda, tkdev, m, k, n, dtype):
    t, want, size = operands(torch_cuda, m * 3 + k + n, m, k, n, whole=False)
    got = f64(product(torch_cuda, tkdev, t, m, k, n, dtype, gap=5 * (m % 2)))
    error = (128 + 3 + -(-k // 128)) * 2.0**-23
    assert (np.abs(got - want) <= error * size + HALF_STEP[dtype] * np.abs(want) + LEAST[dtype]).all()
    if dtype == "f32":
        assert np.linalg.norm(got - want) <= 1e-6 * np.linalg.norm(want)


def test_product_runs_the_same_twice(torch_cuda, tkdev):
    for m, k, n in ((1, 4096, 1024), (48, 2048, 512), (300, 2048, 1024), (1500, 1024, 1500)):
        t, _, _ = operands(torch_cuda, 5, m, k, n, whole=False)
        first = product(torch_cuda, tkdev, t, m, k, n, "f32")
        for _ in range(3):
            assert torch_cuda.equal(first, product(torch_cuda, tkdev, t, m, k, n, "f32"))


@pytest.mark.parametrize("m,n", [(3, 300), (140, 300), (600, 900)])
def test_product_keeps_nan_to_its_rows_and_columns(torch_cuda, tkdev, m, n):
    torch, k = torch_cuda, 700
    t, want, _ = operands(torch, 11, m, k, n, whole=True)
    t[0][1, 600] = 0x7F             # a code of a
    t[1][2, 0] = float("nan")       # a scale of a
    t[2][5, 3] = 0xFF               # a code of w
    t[3][1, 2] = float("inf")       # a scale of w: of columns 128..255
    got = f64(product(torch, tkdev, t, m, k, n, "f32"))
    bad = np.zeros((m, n), bool)
    bad[[1, 2]] = bad[:, 5] = bad[:, 128:256] = True
    assert np.isnan(got[1]).all() and np.isnan(got[2]).all() and np.isnan(got[:, 5]).all()
    assert not np.isfinite(got[bad]).any() and np.array_equal(got[~bad], want[~bad])


def test_product_past_four_gigabytes(torch_cuda, tkdev):
    """Weight and output with more than 2^32 bytes: the last rows of a tall weight, the last row of a wide output."""
    torch, m, k, n = torch_cuda, 3, 128, 34_000_003
    w = torch.zeros((n, k), dtype=torch.uint8, device="cuda")
    at = torch.tensor([0, n // 2, n - 1], device="cuda")
    w[at] = 0x38                                        # 1.0
    t = [torch.full((m, k), 0x38, dtype=torch.uint8, device="cuda"), torch.ones((m, 1), device="cuda"), w,
         torch.ones((-(-n // 128), 1), device="cuda")]
    held = torch.full((m, n), 7.0, device="cuda")
    torch.cuda.synchronize()
    ops.fp8_matmul(tkdev, *t, held, m, k, n)
    want = torch.zeros((m, n), device="cuda")
    want[:, at] = 128.0
    assert torch.equal(held, want)


# ---- as they are used ------------------------------------------------------------------------------

class Block:
    """A projection, the residual's norm, the output head and the choice of tokens, with weights quantised by the
    framework."""

    def __init__(self, torch, dev, rows, hidden, vocab, dtype):
        g = torch.Generator(device="cuda").manual_seed(9)
        t = kind(torch, dtype)
        self.torch, self.dev, self.rows, self.hidden, self.vocab, self.dtype = torch, dev, rows, hidden, vocab, dtype
        empty = lambda *s, d=torch.float32: torch.zeros(s, dtype=d, device="cuda")
        blocks = -(-hidden // 128)
        self.weights = []
        for n in (hidden, vocab):
            w = torch.randn((n, hidden), generator=g, device="cuda") * hidden**-0.5 * 3
            codes, scales = empty(n, hidden, d=torch.uint8), empty(-(-n // 128), blocks)
            torch.cuda.synchronize()
            ops.fp8_quantize(dev, w, codes, scales, n, hidden, 128)
            self.weights.append((codes, scales))
        self.norm = 1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")
        self.x, self.stream_in = empty(rows, hidden, d=t), empty(rows, hidden, d=t)
        self.codes, self.scales = empty(2, rows, hidden, d=torch.uint8), empty(2, rows, blocks)
        self.y, self.logits = empty(rows, hidden, d=t), empty(rows, vocab)
        self.random, self.top_k = empty(rows), torch.full((rows,), 40, dtype=torch.int32, device="cuda")
        self.top_p = torch.full((rows,), 0.9, device="cuda")
        self.tokens, self.kept = (empty(rows, d=torch.int32) for _ in range(2))

    def fill(self, seed):
        g = self.torch.Generator(device="cuda").manual_seed(seed)
        for v in (self.x, self.stream_in):
            v.copy_(self.torch.randn(v.shape, generator=g, device="cuda"))
        self.random.copy_(self.torch.rand(self.rows, generator=g, device="cuda"))

    def step(self, stream):
        q = dict(stream=stream, sync=False)
        r, h, d = self.rows, self.hidden, self.dev
        ops.fp8_quantize(d, self.x, self.codes[0], self.scales[0], r, h, 1, self.dtype, **q)
        ops.fp8_matmul(d, self.codes[0], self.scales[0], *self.weights[0], self.y, r, h, h, self.dtype, **q)
        ops.add_rmsnorm_fp8(d, self.y, self.stream_in, self.norm, self.stream_in, self.codes[1], self.scales[1], r, h, 1e-5,
                            self.dtype, **q)
        ops.fp8_matmul(d, self.codes[1], self.scales[1], *self.weights[1], self.logits, r, h, self.vocab, "f32", **q)
        ops.sample_tokens(d, self.logits, None, self.top_k, self.top_p, None, self.random, self.tokens, self.kept, r,
                          self.vocab, "f32", **q)

    def results(self):
        return [v.clone() for v in (self.y, self.stream_in, self.codes, self.scales, self.logits, self.tokens, self.kept)]


@pytest.mark.parametrize("rows,dtype", [(1, "f32"), (20, "bf16"), (200, "f16")])
def test_a_step_from_attention_to_tokens(torch_cuda, tkdev, rows, dtype):
    """Every output follows, by the oracle, from what the calls before it wrote; captured and replayed with other
    inputs, and run on two streams at once, the bits are the same."""
    torch = torch_cuda
    plain, graphed, other = (Block(torch, tkdev, rows, 768, 5000, dtype) for _ in range(3))
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side[0]):
        graphed.step(side[0].cuda_stream)
    for seed in (1, 2, 3):
        for b in (plain, graphed, other):
            b.fill(seed)
        before = f64(plain.stream_in)
        torch.cuda.synchronize()
        plain.step(1)
        torch.cuda.synchronize()
        graph.replay()
        other.step(side[1].cuda_stream)
        torch.cuda.synchronize()
        for b in (graphed, other):
            assert all(torch.equal(p, q) for p, q in zip(plain.results(), b.results()))
        host = [[v.cpu().numpy() for v in w] for w in plain.weights]
        codes, scales = plain.codes.cpu().numpy(), plain.scales.cpu().numpy()
        y, size = fp8.matmul(codes[0], scales[0], *host[0])
        assert (np.abs(f64(plain.y) - y) <= 140 * 2.0**-23 * size + HALF_STEP[dtype] * np.abs(y) + LEAST[dtype]).all()
        total, normed = fp8.add_rmsnorm(f64(plain.y), before, f64(plain.norm), 1e-5)
        check_codes(normed, codes[1], f64(plain.scales[1]), fp8.group_scales(normed, 1), 1, NORM_ERROR)
        logits, size = fp8.matmul(codes[1], scales[1], *host[1])
        assert (np.abs(f64(plain.logits) - logits) <= 140 * 2.0**-23 * size).all()
        for r, l in enumerate(plain.logits.cpu().numpy()):
            token, kept, slack = fp8.sample(l, None, 40, np.float32(0.9), None, plain.random[r].item())
            assert slack < 1e-9 or (token, kept) == (plain.tokens[r].item(), plain.kept[r].item())
    del graph


def test_calls_leave_the_current_device_and_count_their_launches(torch_cuda, tkdev):
    b = Block(torch_cuda, tkdev, 3, 256, 300, "f32")
    before = tkdev.launch_count()
    b.step(1)
    torch_cuda.cuda.synchronize()
    assert tkdev.launch_count() == before + 5 and torch_cuda.cuda.current_device() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("block", [1, 128])
def test_codes_are_the_nearest_of_the_quotient(torch_cuda, tkdev, block, dtype):
    """Scales are the largest over 448 and codes the conversion of value / scale, bit by bit: 16-bit values over their
    largest lie on ties often."""
    torch = torch_cuda
    x = rows_of(torch, 77, 256, 4096, dtype, 0)
    codes, scales = torch.zeros((256, 4096), dtype=torch.uint8, device="cuda"), torch.zeros((256 // block, 32), device="cuda")
    torch.cuda.synchronize()
    ops.fp8_quantize(tkdev, x, codes, scales, 256, 4096, block, dtype)
    v, s = x.float().cpu(), scales.cpu()
    tiles = v.view(256 // block, block, 32, 128)
    want = tiles.abs().amax((1, 3)) / torch.tensor(448.0)
    assert torch.equal(s, want)
    nearest = (tiles / want[:, None, :, None]).view(256, 4096).to(torch.float8_e4m3fn)
    assert torch.equal(codes.cpu(), nearest.view(torch.uint8))


def test_classes(torch_cuda, tkdev):
    """The objects of kernels.fp8 and kernels.sampler over the framework's own buffers: an odd k, whose rows of codes
    the weight pads."""
    import tiny_kernel as tk
    rng = np.random.default_rng(5)
    m, k, n = 4, 300, 500
    x, r, weight = rng.normal(size=(m, k)), rng.normal(size=(m, k)), 1 + 0.1 * rng.normal(size=k)
    w = rng.normal(size=(n, k)) * k**-0.5
    buf = lambda a: tkdev.create_buffer_with_data("f32", np.asarray(a, np.float32))
    new = lambda t, c: tkdev.create_buffer(t, c)
    fp = tk.kernels.fp8
    linear = fp.LinearFP8.init(tkdev, n, k)
    linear.load(buf(w))
    total, codes, scales = new("f32", m * k), new("u8", m * k), new("f32", m * fp.blocks(k))
    fp.AddRMSNormFP8.init(tkdev).forward(buf(x), buf(r), buf(weight), total, codes, scales, k, 1e-5)
    want_sum, y = fp8.add_rmsnorm(x.astype(np.float32), r.astype(np.float32), weight.astype(np.float32), 1e-5)
    check_codes(y, codes.read().reshape(m, k), scales.read().reshape(m, -1).astype(np.float64), fp8.group_scales(y, 1), 1, NORM_ERROR)
    assert np.abs(total.read().reshape(m, k) - want_sum).max() <= 2.0**-23 * np.abs(want_sum).max()
    again, scales2 = new("u8", m * k), new("f32", m * fp.blocks(k))
    fp.QuantizeFP8.init(tkdev).forward(total, again, scales2, k)
    padded = tkdev.create_buffer_with_data("u8", np.pad(again.read().reshape(m, k), ((0, 0), (0, linear.row - k))))
    logits = new("f32", m * n)
    linear.forward(padded, scales2, logits, m, a_stride=linear.row)
    want, size = fp8.matmul(again.read().reshape(m, k), scales2.read().reshape(m, -1), linear.codes.read().reshape(n, -1)[:, :k],
                            linear.scales.read().reshape(fp.blocks(n), -1))
    assert (np.abs(logits.read().reshape(m, n) - want) <= 140 * 2.0**-23 * size).all()
    tokens, kept = new("i32", m), new("i32", m)
    u = np.array([0.1, 0.4, 0.6, 0.9], np.float32)
    tk.kernels.sampler.SampleTokens.init(tkdev).forward(logits, None, None, buf([0.9] * m), None, buf(u), tokens, kept)
    for i, l in enumerate(logits.read().reshape(m, n)):
        token, count, slack = fp8.sample(l, None, None, np.float32(0.9), None, u[i])
        assert slack < 1e-9 or (token, count) == (tokens.read()[i], kept.read()[i])
    linear.deinit()


def test_as_many_rows_as_a_call_takes(torch_cuda, tkdev):
    """Rows of one value, each a group of its own: more groups than 2^32 threads have, and the largest number of rows."""
    torch = torch_cuda
    rows = 2**28 + 37
    x = torch.arange(rows, dtype=torch.float32, device="cuda") % 97 + 1
    codes, scales = torch.zeros(rows, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ops.fp8_quantize(tkdev, x, codes, scales, rows, 1)
    assert (codes == 0x7E).all() and torch.equal(scales, x / torch.tensor(448.0, device="cuda"))
    del x, codes, scales
    rows = 2**31 - 1
    x = torch.full((rows,), -3.0, dtype=torch.bfloat16, device="cuda")
    codes, scales = torch.zeros(rows, dtype=torch.uint8, device="cuda"), torch.zeros(rows, device="cuda")
    torch.cuda.synchronize()
    ops.add_rmsnorm_fp8(tkdev, x, None, None, None, codes, scales, rows, 1, 0.0, "bf16")
    assert codes.min().item() == codes.max().item() == 0xFE
    assert abs(scales.min().item() * 448 - 1) < 1e-6 and abs(scales.max().item() * 448 - 1) < 1e-6
