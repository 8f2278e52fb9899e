"""GPU parity of the serving-step operators over the 4-bit key/value cache (tk_paged_slots,
tk_qk_norm_rope, tk_kv4_append, tk_kv4_gather, tk_kv4_attention) against the f64 oracle.

Whole numbers, codes, scales and values read back are equal.  Norm and rotation: every value within
32 * 2^-24 of the size of its pair (the sum of squares rounds at most D/32 + 8 times and its square
root halves that, eight roundings follow; D <= 512 here) and half a step of its type.  Attention:
the oracle's bound of f32 sums per value, and 1e-5 of the largest output as for the f32 cache, each
with half a step of the output's type.
"""
import numpy as np
import pytest

import kv4 as oracle4
from tiny_kernel import _lib, ops

pytestmark = pytest.mark.gpu

HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
LEAST = {"f32": 0.0, "f16": 2.0**-25, "bf16": 0.0}  # half the least step of f16


def kind(torch, name):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def i32(torch, a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def f64(t):
    return t.double().cpu().numpy()


# ---- block tables and slots ----------------------------------------------------------------------

SLOTS = [
    # ctx, new, block_size, spare table width, pages in the list beyond the need, spare tokens
    ([0], [1], 16, 0, 0, 0),
    ([15, 16, 17], [1, 1, 1], 16, 2, 3, 5),
    ([0, 31, 0, 64], [33, 0, 1, 64], 32, 1, 0, 3),
    ([5, -3, 0, 100], [-1, 4, 0, 60], 16, 0, 2, 9),
    ([0, 0, 0], [0, 0, 0], 64, 0, 1, 4),
    ([3] * 300, [1] * 300, 16, 0, 1, 0),                      # more requests than threads
    ([7 * i % 50 for i in range(1000)], [i % 23 for i in range(1000)], 16, 1, 4, 77),
    ([0, 1000], [5000, 3000], 256, 0, 0, 1),
    ([10, 10, 10], [30, 30, 30], 16, 0, -3, 0),               # the pool runs out
    ([10, 40], [50, 70], 16, -3, 5, 2),                       # the table is too narrow
    ([10, 5, 9], [50, 70, 20], 16, 0, 0, -60),                # more tokens than rows
    ([2**31 - 3], [10], 256, -8388600, 0, 3),                 # positions end at the int's end
]


def slots_case(seed, ctx, new, bs, width, pool, tokens):
    rng = np.random.default_rng(seed)
    c, n = np.maximum(ctx, 0).astype(np.int64), np.maximum(new, 0).astype(np.int64)
    n = np.minimum(n, 2**31 - 1 - c)
    have, need = -(-c // bs), -(-(c + n) // bs)
    width = max(1, int(need.max()) + width)
    have, need = np.minimum(have, width), np.minimum(need, width)
    blocks = int(need.sum()) + max(pool, 0) + 2
    order = rng.permutation(blocks).astype(np.int32)
    tables = np.full((len(ctx), width), -1, np.int32)
    at = 0
    for b, h in enumerate(have):
        tables[b, :h] = order[at:at + h]
        at += h
    count = int((need - have).sum()) + pool
    free = np.concatenate([[-7, -7], order[at:at + max(count, 0)]]).astype(np.int32)
    return (np.array(ctx), np.array(new), free, np.array([2, 2 + max(count, 0)]), tables, bs, blocks,
            max(1, int(n.sum()) + tokens))


def run_slots(torch, dev, case, stream=None):
    ctx, new, free, rng, tables, bs, blocks, tokens = case
    t = i32(torch, tables)
    batch = len(ctx)
    out = [torch.full((m,), -99, dtype=torch.int32, device="cuda") for m in (batch, batch + 1, tokens, tokens, 4)]
    args = [i32(torch, x) for x in (ctx, new, free, rng)]
    torch.cuda.synchronize()
    ops.paged_slots(dev, *args, t, *out, batch, tables.shape[1], bs, blocks, tokens)
    return [x.cpu().numpy() for x in [t] + out]


@pytest.mark.parametrize("n", range(len(SLOTS)))
def test_paged_slots(torch_cuda, tkdev, n):
    case = slots_case(n, *SLOTS[n])
    want = oracle4.paged_slots(*case)
    for name, x, y in zip("tables kv_lens query_start positions slots counts".split(),
                          run_slots(torch_cuda, tkdev, case), want):
        assert np.array_equal(x, y), name


def test_paged_slots_ids_outside_the_cache(torch_cuda, tkdev):
    """Ids outside the cache, in the tables and in the free list, give no slot and are counted."""
    case = list(slots_case(3, [20, 40, 3], [30, 30, 30], 16, 1, 2, 0))
    case[2][[3, 4]] = [case[6], -5]          # two of the free list
    case[4][1, 2] = case[6] + 3              # the page that request 1 has begun
    want = oracle4.paged_slots(*case)
    assert want[5][2] > 0
    for x, y in zip(run_slots(torch_cuda, tkdev, case), want):
        assert np.array_equal(x, y)


# ---- norms and rotation --------------------------------------------------------------------------

QK = [
    # tokens, q_heads, kv_heads, dim, rot, interleaved, norm, gap (elements between rows), offset
    (1, 32, 8, 128, 128, False, True, 0, 0),
    (5, 14, 2, 64, 64, False, True, 0, 0),
    (7, 3, 3, 128, 64, True, False, 24, 0),
    (3, 8, 1, 256, 128, False, True, 0, 0),
    (2, 5, 0, 128, 128, False, True, 0, 0),
    (4, 0, 3, 64, 32, True, True, 0, 0),
    (6, 4, 2, 80, 80, False, True, 0, 0),     # a dimension of its own kernel
    (3, 2, 1, 96, 48, True, True, 3, 0),
    (3, 2, 1, 6, 2, False, True, 0, 0),
    (2, 1, 1, 512, 100, False, False, 0, 0),
    (9, 4, 2, 128, 0, False, True, 0, 0),     # the norm alone
    (9, 4, 2, 128, 36, False, True, 0, 0),    # half of it no whole load
    (5, 4, 2, 128, 128, False, True, 1, 1),   # rows on no 16-byte boundary
    (300, 9, 3, 64, 64, False, False, 8, 0),
    (4, 5, 2, 48, 48, False, True, 8, 0),     # lanes that hold nothing
    (3, 5, 2, 96, 32, False, True, 0, 0),
    (5, 2, 2, 160, 20, True, True, 0, 0),     # a lane's values turned in part
    (2, 3, 2, 256, 256, False, True, 4, 4),
    (700, 18, 3, 128, 128, False, True, 0, 0),  # groups of heads, the last not full
    (800, 9, 6, 112, 56, True, False, 0, 0),
]


def qk_case(torch, seed, tokens, hq, hk, dim, rot, norm, dtype, gap, offset):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    row, far = (hq + hk) * dim + gap, 50
    flat = torch.randn(tokens * row + offset, generator=gen, device="cuda").to(kind(torch, dtype))
    x = flat[offset:].view(tokens, row)
    turn = torch.rand((far, max(rot // 2, 1)), generator=gen, device="cuda") * 6.3
    w = [1 + 0.2 * torch.randn(dim, generator=gen, device="cuda") if norm else None for _ in range(2)]
    pos = torch.randint(0, far, (tokens,), generator=gen, device="cuda", dtype=torch.int32)
    return x, w, turn.cos(), turn.sin(), pos, far, row


def check_qk(y, x, w, cos, sin, pos, rot, interleaved, dtype):
    want, size = oracle4.qk_norm_rope_f64(f64(x), None if w is None else f64(w), f64(cos), f64(sin),
                                          pos.cpu().numpy(), rot, interleaved, 1e-5)
    off = np.abs(f64(y) - want)
    assert (off <= 32 * 2.0**-24 * size * (1 + HALF_STEP[dtype]) + HALF_STEP[dtype] * np.abs(want) + LEAST[dtype]).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", range(len(QK)))
def test_qk_norm_rope(torch_cuda, tkdev, n, dtype):
    torch = torch_cuda
    tokens, hq, hk, dim, rot, inter, norm, gap, offset = QK[n]
    x, w, cos, sin, pos, far, row = qk_case(torch, n, tokens, hq, hk, dim, rot, norm, dtype, gap, offset)
    q, k = x[:, :hq * dim], x[:, hq * dim:(hq + hk) * dim]
    qo, ko = torch.empty_like(q), torch.empty_like(k)   # rows as far apart as the inputs'
    qo, ko = (torch.full((tokens, m * dim), float("nan"), dtype=x.dtype, device="cuda") for m in (hq, hk))
    torch.cuda.synchronize()
    ops.qk_norm_rope(tkdev, q, k, *w, cos, sin, pos, qo, ko, tokens, hq, hk, dim, rot, far, 1e-5, dtype,
                     interleaved=inter, q_stride=row, k_stride=row)
    for y, v, m, wt in ((qo, q, hq, w[0]), (ko, k, hk, w[1])):
        if m:
            check_qk(y.view(tokens, m, dim), v.unflatten(1, (m, dim)), wt, cos, sin, pos, rot, inter, dtype)


@pytest.mark.parametrize("dim,rot", [(128, 128), (80, 40)])
def test_qk_norm_rope_in_place_leaves_padding(torch_cuda, tkdev, dim, rot):
    """In place, with tokens whose position is outside the cache of angles: their rows stay."""
    torch = torch_cuda
    x, w, cos, sin, pos, far, row = qk_case(torch, 5, 9, 4, 2, dim, rot, True, "f32", 8, 0)
    before = x.clone()
    good = pos.clone()
    pos[[1, 4, 8]] = torch.tensor([-1, far, 2**31 - 1], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ops.qk_norm_rope(tkdev, x, x[:, 4 * dim:], *w, cos, sin, pos, x, x[:, 4 * dim:], 9, 4, 2, dim, rot, far, 1e-5,
                     q_stride=row, k_stride=row, q_out_stride=row, k_out_stride=row)
    assert torch.equal(x[[1, 4, 8]], before[[1, 4, 8]]) and torch.equal(x[:, 6 * dim:], before[:, 6 * dim:])
    on = [0, 2, 3, 5, 6, 7]
    for a, m, wt in ((0, 4, w[0]), (4, 2, w[1])):
        part = [t[on][:, a * dim:(a + m) * dim].reshape(6, m, dim) for t in (x, before)]
        check_qk(part[0], part[1], wt, cos, sin, good[on], rot, False, "f32")


def test_qk_norm_rope_keeps_what_is_not_finite_in_its_head(torch_cuda, tkdev):
    torch = torch_cuda
    x, w, cos, sin, pos, far, row = qk_case(torch, 6, 2, 3, 1, 128, 64, False, "f32", 0, 0)
    x[0, 130] = float("inf")
    x[1, 100] = float("nan")
    out = torch.zeros((2, 3 * 128), device="cuda")
    ko = torch.zeros((2, 128), device="cuda")
    torch.cuda.synchronize()
    ops.qk_norm_rope(tkdev, x, x[:, 384:], None, None, cos, sin, pos, out, ko, 2, 3, 1, 128, 64, far, 1e-5,
                     q_stride=row, k_stride=row)
    odd = ~torch.isfinite(out)
    # a pair of the infinity; past the rotated part a value stays as it is
    assert odd[0].nonzero().flatten().tolist() == [130, 162] and odd[1].nonzero().flatten().tolist() == [100]


# ---- quantised writes and reads ------------------------------------------------------------------

def new_cache(torch, blocks, hk, bs, dim, group, fill=0):
    codes = [torch.full((blocks, hk, bs, dim // 2), fill, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.full((blocks, hk, bs, dim // group, 2), 0.25, dtype=torch.float16, device="cuda") for _ in range(2)]
    return codes + scales, ops.kv4_cache(*codes, *scales, blocks, hk, bs, dim, group)


WRITES = [(1, 1, 64, 64, 16), (5, 2, 128, 128, 16), (33, 3, 128, 64, 32), (70, 1, 256, 64, 64),
          (19, 5, 256, 128, 128), (40, 2, 64, 64, 256)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,hk,dim,group,bs", WRITES)
def test_append_and_gather(torch_cuda, tkdev, tokens, hk, dim, group, bs, dtype):
    torch = torch_cuda
    gen = torch.Generator(device="cuda").manual_seed(tokens)
    row = hk * dim
    kv = (torch.randn((tokens, 2 * row + 8), generator=gen, device="cuda") * 5).to(kind(torch, dtype))
    kv[0, :group] = 1.5                      # a group of one value
    kv[-1, -8 - group:-8] *= 1e-4            # a small one
    k, v = kv[:, :row], kv[:, row:2 * row]
    blocks = -(-tokens // bs) + 3
    bufs, cache = new_cache(torch, blocks, hk, bs, dim, group, 0xA5)
    slots = torch.randperm(blocks * bs, generator=gen, device="cuda")[:tokens].to(torch.int32)
    drop = tokens // 2 if tokens > 2 else -1
    if drop >= 0:
        slots[drop] = -1
    before = [b.clone() for b in bufs]
    stride = kv.shape[1]
    back = torch.full((tokens, 2 * row), 77.0, dtype=kv.dtype, device="cuda")
    torch.cuda.synchronize()
    ops.kv4_append(tkdev, cache, k, v, slots, tokens, dtype, k_stride=stride, v_stride=stride)
    ops.kv4_gather(tkdev, cache, slots, back, back[:, row:], tokens, dtype, k_stride=2 * row, v_stride=2 * row)
    s = slots.long()
    on = s >= 0
    page, at = s[on] // bs, s[on] % bs
    for x, codes, scales, b in ((k, bufs[0], bufs[2], back[:, :row]), (v, bufs[1], bufs[3], back[:, row:])):
        c, sc, of = oracle4.quantise(f64(x[on]).reshape(-1, hk, dim), group)
        assert np.array_equal(codes[page, :, at].cpu().numpy(), oracle4.pack(c))
        assert np.array_equal(scales[page, :, at].cpu().numpy(), np.stack((sc, of), -1))
        want = torch.from_numpy(oracle4.values_f64(c, sc, of)).float().to(kv.dtype)  # exact in f32
        assert torch.equal(b[on].cpu().view(-1, hk, dim), want)
        if drop >= 0:
            assert (b[drop] == 77).all()
    for b, old in zip(bufs, before):         # the other slots stay
        b[page, :, at] = old[page, :, at]
        assert torch.equal(b, old)


def test_append_ties_go_to_the_even_code(torch_cuda, tkdev):
    """Quotients on and next to .5 (f32 neighbours of a tie): the true quotient decides."""
    torch = torch_cuda
    x = np.zeros((1, 1, 64), np.float32)
    x[0, 0, 1] = 15 * 0.75
    for i in range(15):
        tie = np.float32((i + 0.5) * 0.75)
        x[0, 0, 2 + 4 * i:6 + 4 * i] = [tie, np.nextafter(tie, np.float32(99)), np.nextafter(tie, np.float32(-99)), i]
    t = torch.from_numpy(x).cuda()
    slots = i32(torch, [3])
    bufs, cache = new_cache(torch, 1, 1, 16, 64, 64)
    torch.cuda.synchronize()
    ops.kv4_append(tkdev, cache, t, t, slots, 1)
    c, _, _ = oracle4.quantise(x, 64)
    assert np.array_equal(oracle4.unpack(bufs[0][0, 0, 3].cpu().numpy()), c[0, 0])
    # thirds: the f32 quotient itself falls on ties that the true one misses
    y = (np.random.default_rng(9).integers(0, 2**24, (4096, 1, 64)) / 2.0**22).astype(np.float32)
    bufs, cache = new_cache(torch, 256, 1, 16, 64, 64)
    t = torch.from_numpy(y).cuda()
    slots = torch.arange(4096, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ops.kv4_append(tkdev, cache, t, t, slots, 4096)
    assert np.array_equal(bufs[1].cpu().numpy().reshape(4096, 32), oracle4.pack(oracle4.quantise(y, 64)[0]).reshape(4096, 32))


def test_append_of_large_and_not_finite_values(torch_cuda, tkdev):
    torch = torch_cuda
    x = torch.randn((4, 1, 128), device="cuda")
    x[0, 0, 3], x[0, 0, 70] = 3e38, -3e38       # saturates
    x[1, 0, 3] = float("nan")
    x[2, 0, 100] = float("inf")
    x[3, 0, :64] = float("-inf")
    bufs, cache = new_cache(torch, 1, 1, 16, 128, 64)
    slots = i32(torch, [0, 1, 2, 3])
    back = torch.zeros((2, 4, 1, 128), device="cuda")
    torch.cuda.synchronize()
    ops.kv4_append(tkdev, cache, x, x, slots, 4)
    ops.kv4_gather(tkdev, cache, slots, back[0], back[1], 4)
    assert torch.equal(torch.isnan(back[0]).view(4, 2, 64).any(-1).cpu(),
                       torch.tensor([[False, False], [True, False], [False, True], [True, False]]))
    assert torch.equal(torch.isnan(back[0]).view(4, 2, 64).all(-1), torch.isnan(back[0]).view(4, 2, 64).any(-1))
    c, s, m = oracle4.quantise(f64(x), 64)
    assert np.array_equal(bufs[2][0, 0, :4].cpu().numpy(), np.stack((s, m), -1)[:, 0], equal_nan=True)
    assert np.array_equal(oracle4.unpack(bufs[0][0, 0, :4].cpu().numpy()), c[:, 0])


def test_slots_outside_the_cache_are_ignored(torch_cuda, tkdev):
    torch = torch_cuda
    x = torch.randn((4, 2, 64), device="cuda")
    bufs, cache = new_cache(torch, 3, 2, 16, 64, 64, 0x5A)
    before = [b.clone() for b in bufs]
    slots = i32(torch, [48, -1, 2**31 - 1, -2**31])
    back = torch.full((2, 4, 2, 64), 5.0, device="cuda")
    torch.cuda.synchronize()
    ops.kv4_append(tkdev, cache, x, x, slots, 4)
    ops.kv4_gather(tkdev, cache, slots, back[0], back[1], 4)
    assert all(torch.equal(a, b) for a, b in zip(bufs, before)) and (back == 5).all()


# ---- attention -----------------------------------------------------------------------------------

class Case:
    """A cache filled at random, tables of shuffled pages, ragged queries."""

    def __init__(self, torch, seed, kv_lens, queries, hq, hk, dim, group, bs, dtype, spare=2, size=1.0):
        rng = np.random.default_rng(seed)
        self.torch, self.bs, self.dtype, self.hq, self.hk, self.dim = torch, bs, dtype, hq, hk, dim
        pages = [-(-max(n, 1) // bs) for n in kv_lens]
        self.width, self.blocks = max(pages) + spare, sum(pages) + 3
        order = rng.permutation(self.blocks)
        self.tables = np.full((len(kv_lens), self.width), -1, np.int32)
        at = 0
        for b, n in enumerate(pages):
            self.tables[b, :n] = order[at:at + n]
            at += n
        shape = (self.blocks, hk, bs, dim)
        self.parts = []
        for _ in range(2):
            codes = rng.integers(0, 16, shape).astype(np.uint8)
            scale = (0.3 * np.exp(0.5 * rng.standard_normal(shape[:3] + (dim // group,)))).astype(np.float16)
            offset = (-7.5 * scale.astype(np.float64) * (1 + 0.2 * rng.standard_normal(scale.shape))).astype(np.float16)
            self.parts.append([codes, scale, offset])
        self.kv_lens = np.array(kv_lens, np.int32)
        self.start = None if queries is None else np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
        self.tokens = len(kv_lens) if queries is None else int(self.start[-1])
        q = torch.from_numpy(rng.standard_normal((max(self.tokens, 1), hq, dim)) * size)
        self.q = q.to(kind(torch, dtype)).cuda()
        self.scale = dim ** -0.5

    def upload(self):
        bufs = []
        for i in range(2):
            bufs.append(self.torch.from_numpy(oracle4.pack(self.parts[i][0])).cuda())
        for i in range(2):
            bufs.append(self.torch.from_numpy(np.stack(self.parts[i][1:], -1)).cuda())
        self.bufs = bufs
        group = self.dim // self.parts[0][1].shape[-1]
        return ops.kv4_cache(*bufs, self.blocks, self.hk, self.bs, self.dim, group)

    def want(self):
        (kc, ks, ko), (vc, vs, vo) = self.parts
        zero = np.zeros_like(ko)
        centre = vo.astype(np.float64) + 8 * vs.astype(np.float64)
        v_size = oracle4.values_f64(np.full_like(vc, 8), vs, zero) + oracle4.values_f64(
            np.zeros_like(vc), vs, np.abs(centre))
        k_size = oracle4.values_f64(kc, ks, np.abs(ko.astype(np.float64)))
        return oracle4.attention_f64(f64(self.q), oracle4.values_f64(kc, ks, ko), oracle4.values_f64(vc, vs, vo), k_size,
                                     v_size, self.tables, self.kv_lens, self.start, self.scale, self.bs)

    def run(self, dev, cache, o=None, stream=None):
        torch = self.torch
        self.o = torch.full_like(self.q, 55.0) if o is None else o
        self.ws_size = ops.kv4_attention_workspace(dev, cache, self.hq)
        self.ws = torch.full((self.ws_size,), 0xFF, dtype=torch.uint8, device="cuda")
        self.dev_args = [i32(torch, self.tables), i32(torch, self.kv_lens),
                         None if self.start is None else i32(torch, self.start)]
        torch.cuda.synchronize()
        ops.kv4_attention(dev, cache, self.q, *self.dev_args, self.o, self.ws, self.ws_size, self.tokens,
                          len(self.kv_lens), self.hq, self.width, self.scale, self.dtype, stream=stream)
        return self.o

    def check(self, o, rows=slice(None)):
        want, bound = self.want()
        y, want, bound = f64(o)[rows], want[rows], bound[rows]
        assert np.isfinite(want).all()
        off, step = np.abs(y - want), HALF_STEP[self.dtype]
        assert (off <= bound * (1 + step) + step * np.abs(want) + LEAST[self.dtype]).all()
        assert off.max() <= (1e-5 + step) * np.abs(want).max() if want.size and want.any() else not y.any()


ATTENTION = [
    # kv_lens, queries (None: one each), q_heads, kv_heads, dim, group, block_size
    ([1], None, 1, 1, 64, 64, 16),
    ([16, 17, 15], None, 4, 2, 128, 128, 16),
    ([500], None, 32, 8, 128, 128, 16),
    ([0, 3, 0, 70], None, 8, 1, 128, 64, 32),             # contexts with nothing in them
    ([333, 1, 64, 129], None, 16, 2, 256, 128, 64),
    ([2100, 30], None, 10, 2, 128, 128, 16),              # five query heads a key head
    ([255, 257], None, 16, 1, 64, 64, 256),
    ([40, 41], None, 3, 3, 256, 64, 16),
    ([300, 77, 5], [5, 1, 3], 8, 2, 64, 64, 64),          # drafted tokens
    ([100, 20, 64], [0, 20, 64], 6, 2, 128, 64, 16),      # no query; whole prompts
    ([50, 2, 0], [17, 6, 2], 4, 4, 128, 128, 16),         # queries before the first position
    ([700, 130], [130, 33], 7, 1, 128, 128, 32),
    ([1, 0], [1, 1], 2, 2, 64, 64, 16),
    ([4000], [3], 12, 4, 256, 64, 128),
    ([37] * 70, None, 4, 4, 64, 64, 16),
    ([5000] + [20] * 150, None, 8, 2, 128, 128, 16),      # one long, many short
    ([90] + [17] * 29, [30] + [1] * 29, 4, 2, 128, 64, 16),  # one token on the mean, thirty once
    ([260, 31, 7], [1, 0, 2], 4, 1, 64, 64, 32),          # four heads a group: one row a head
    ([1500], [1], 3, 1, 256, 128, 16),
    ([10, 700], None, 2, 1, 128, 64, 64),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", range(len(ATTENTION)))
def test_attention(torch_cuda, tkdev, n, dtype):
    c = Case(torch_cuda, n, *ATTENTION[n], dtype)
    c.check(c.run(tkdev, c.upload()))


# many rows a sequence, a long table: the kernel for prompts (f32: where there are 64 rows on the mean)
PROMPTS = [
    ([128], [128], 1, 1, 128, 128, 16),                      # one full tile, one step
    ([1], [1], 50, 1, 64, 64, 16),                           # one token in all
    ([129, 300], [129, 33], 4, 4, 64, 64, 16),               # a row and a step more than full ones
    ([700, 130], [130, 33], 7, 1, 128, 128, 32),
    ([1000, 17, 0, 400], [100, 17, 0, 1], 10, 2, 128, 128, 64),  # a prompt, one token, no request
    ([50, 2, 0, 9], [60, 40, 3, 9], 16, 8, 128, 128, 16),    # queries before the first position
    ([2500], [70], 16, 1, 64, 64, 256),                      # many CTAs to a tile
    ([300] * 20, [50] * 20, 4, 4, 64, 64, 16),
    ([5200] * 4, [130] * 4, 16, 16, 64, 64, 32),             # runs long enough for sums to be set aside
    ([4600, 4300, 4400], [257, 256, 140], 10, 10, 128, 128, 16),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", range(len(PROMPTS)))
def test_attention_of_prompts(torch_cuda, tkdev, n, dtype):
    c = Case(torch_cuda, 40 + n, *PROMPTS[n], dtype, spare=6000)
    c.check(c.run(tkdev, c.upload()))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 128)])
def test_attention_of_prompts_in_every_form(torch_cuda, tkdev, dim, group, dtype):
    c = Case(torch_cuda, 81, [900, 17, 0, 300], [129, 17, 0, 40], 9, 3, dim, group, 32, dtype, spare=100)
    c.check(c.run(tkdev, c.upload()))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim,group,hk", [(128, 64, 20), (128, 128, 12), (256, 64, 8), (256, 128, 8)])
def test_long_prompts_set_their_sums_aside(torch_cuda, tkdev, dim, group, hk, dtype):
    """Runs of more steps than the sums of the tensor core are left to themselves."""
    c = Case(torch_cuda, 82, [5000] * 3, [161] * 3, hk, hk, dim, group, 16, dtype)
    c.check(c.run(tkdev, c.upload()))


@pytest.mark.parametrize("dim,group,dtype", [(64, 64, "f16"), (128, 128, "f16"), (128, 64, "f32"), (256, 64, "bf16")])
def test_prompts_with_absent_pages_and_anything_in_masked_places(torch_cuda, tkdev, dim, group, dtype):
    """Pages that are not in the cache (more than a step of them, and the whole of a sequence), and
    NaN and infinities in scales behind the last token, in pages of nobody and in the last query's own
    position, which only it sees."""
    c = Case(torch_cuda, 61, [700, 2500, 40], [100, 40, 40], 4, 2, dim, group, 16, dtype, spare=6000)
    c.tables[0, 3:14] = -1
    c.tables[1, :140] = c.blocks
    c.tables[2, :] = [-5, 2**31 - 1, -2**31] + [-1] * (c.width - 3)
    for part in c.parts:
        for b, n in enumerate(c.kv_lens):
            page = c.tables[b, n // 16]
            if 0 <= page < c.blocks:
                part[1][page, :, n % 16:], part[2][page, :, n % 16:] = np.nan, np.inf
        part[1][np.setdiff1d(np.arange(c.blocks), c.tables)] = np.inf
    o = c.run(tkdev, c.upload())
    c.check(o)
    assert not o[140:].any()
    last = c.tables[0, 699 // 16]
    c.parts[1][1][last, :, 699 % 16] = np.inf
    c.parts[0][2][last, :, 699 % 16] = np.nan
    p = c.run(tkdev, c.upload())
    assert torch_cuda.isnan(p[99]).all() and torch_cuda.equal(p[:99], o[:99]) and torch_cuda.equal(p[100:], o[100:])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompts_in_place_strided_and_repeated(torch_cuda, tkdev, dtype):
    """Rows of a projection apart and off the 16-byte boundary, output over the queries; the same bits
    from run to run, and rows of no sequence left as they were."""
    torch = torch_cuda
    c = Case(torch, 62, [900, 333], [90, 40], 6, 2, 64, 64, 16, dtype, spare=6000)
    cache = c.upload()
    first = c.run(tkdev, cache).clone()
    for _ in range(3):
        assert torch.equal(c.run(tkdev, cache), first)
    wide = torch.full((135, 6 * 64 + 3), 9.0, dtype=c.q.dtype, device="cuda")
    wide[2:132, 1:385] = c.q.view(130, 384)
    c.dev_args[2] = i32(torch, [2, 92, 132])
    row = wide[:, 1:]
    torch.cuda.synchronize()
    ops.kv4_attention(tkdev, cache, row, *c.dev_args, row, c.ws, c.ws_size, 135, 2, 6, c.width, c.scale, dtype,
                      q_stride=387, o_stride=387)
    assert torch.equal(wide[2:132, 1:385], first.view(130, 384))
    wide[2:132, 1:385] = 9
    assert (wide == 9).all()


@pytest.mark.parametrize("dtype,group,spare", [("f16", 128, 6000), ("bf16", 128, 6000), ("f32", 128, 6000),
                                               ("bf16", 64, 6000), ("f32", 128, 2), ("f32", 64, 2), ("bf16", 64, 2)])
def test_prompts_with_scales_of_every_kind(torch_cuda, tkdev, dtype, group, spare):
    """Scales of 0, of either sign, the smallest subnormal and sizes far apart; queries of every size;
    a row of queries with an infinity gives NaN and no other row does."""
    c = Case(torch_cuda, 63, [600, 200], [64, 40], 2, 1, 128, group, 16, dtype, spare=spare)
    rng = np.random.default_rng(63)
    for part in c.parts:
        some = rng.integers(0, 8, part[1].shape)
        part[1][some == 0] = 0
        part[1][some == 1] *= -1
        part[1][some == 2] = 2.0**-24
        part[1][some == 3] *= np.float16(2.0**-9)
        part[2][some == 2] = 0.25
    c.q[::7] *= 1e-3
    c.q[::11] *= 6
    o = c.run(tkdev, c.upload()).clone()
    c.check(o)
    c.q[70, 1, 5] = float("inf")
    p = c.run(tkdev, c.upload())
    assert torch_cuda.isnan(p[70, 1]).all()
    p[70, 1] = o[70, 1]
    assert torch_cuda.equal(p, o)


def test_attention_repeats_bit_for_bit(torch_cuda, tkdev):
    c = Case(torch_cuda, 3, [3000, 17, 900], [1, 4, 2], 8, 2, 128, 128, 16, "f32")
    cache = c.upload()
    first = c.run(tkdev, cache).clone()
    for _ in range(3):
        assert torch_cuda.equal(c.run(tkdev, cache), first)


def test_attention_pages_outside_the_cache_are_absent(torch_cuda, tkdev):
    c = Case(torch_cuda, 4, [90, 40, 33], None, 4, 2, 128, 128, 16, "f32")
    c.tables[0, 2], c.tables[0, 4] = -1, c.blocks
    c.tables[1, :] = [-5, 2**31 - 1, -2**31] + [c.blocks] * (c.width - 3)   # nothing of it is there
    o = c.run(tkdev, c.upload())
    c.check(o)
    assert not o[1].any()


def test_attention_masked_places_may_hold_anything(torch_cuda, tkdev):
    """Scales of NaN and infinity behind the last token of a page, in unused pages and at positions
    that a query does not see do not reach the outputs; a NaN that it sees does."""
    c = Case(torch_cuda, 5, [37, 20], [3, 1], 4, 2, 128, 64, 16, "f32")
    for part in c.parts:
        for b, n in enumerate(c.kv_lens):
            page = c.tables[b, n // 16]
            part[1][page, :, n % 16:] = np.nan
            part[2][page, :, n % 16:] = np.inf
        part[1][np.setdiff1d(np.arange(c.blocks), c.tables)] = np.inf
    clean = Case(torch_cuda, 5, [37, 20], [3, 1], 4, 2, 128, 64, 16, "f32")
    clean.check(c.run(tkdev, c.upload()))
    page = c.tables[0, 36 // 16]
    c.parts[1][1][page, :, 36 % 16] = np.nan     # the value at the last position: the last query's alone
    c.parts[0][2][page, 0, 36 % 16] = -np.inf
    o = c.run(tkdev, c.upload())
    clean.check(o, [0, 1, 3])
    assert torch_cuda.isnan(o[2]).all()


def test_attention_rows_of_no_sequence_stay(torch_cuda, tkdev):
    """A padded step: rows before, between and behind the sequences; and o may be q."""
    torch = torch_cuda
    c = Case(torch, 6, [64, 30], [2, 4], 4, 1, 64, 64, 16, "f32")
    c.q = torch.randn((12, 4, 64), device="cuda")
    c.tokens = 12
    c.start = np.array([3, 5, 9], np.int32)
    o = c.run(tkdev, c.upload())
    out = [0, 1, 2, 9, 10, 11]
    assert (o[out] == 55).all()
    c.check(o, slice(3, 9))
    q = c.q.clone()
    c2 = Case(torch, 6, [64, 30], [2, 4], 4, 1, 64, 64, 16, "f32")
    c2.q, c2.tokens, c2.start = q, 12, c.start
    got = c2.run(tkdev, c2.upload(), o=q)
    assert torch.equal(got[3:9], o[3:9]) and torch.equal(got[out], c.q[out])


def test_attention_strided_rows(torch_cuda, tkdev):
    torch = torch_cuda
    c = Case(torch, 7, [100, 33], None, 4, 2, 128, 128, 16, "bf16")
    wide = torch.zeros((2, 4 * 128 + 40), dtype=torch.bfloat16, device="cuda")
    wide[:, 5:5 + 512] = c.q.view(2, 512)
    out = torch.full((2, 4 * 128 + 7), 9.0, dtype=torch.bfloat16, device="cuda")
    cache = c.upload()
    want = c.run(tkdev, cache)
    ops.kv4_attention(tkdev, cache, wide[:, 5:], *c.dev_args, out, c.ws, c.ws_size, 2, 2, 4, c.width, c.scale, "bf16",
                      q_stride=552, o_stride=519)
    assert torch.equal(out[:, :512], want.view(2, 512)) and (out[:, 512:] == 9).all()


def test_attention_scales_far_apart(torch_cuda, tkdev):
    """Value scales from f16's least to its largest, large scores, a zero and a negative scale."""
    torch = torch_cuda
    for seed, scale, spread in ((8, 0.09, 8.0), (9, -0.2, 0.0), (10, 0.0, 3.0), (11, 3.0, 1.0)):
        c = Case(torch, seed, [150], None, 4, 2, 128, 64, 16, "f32")
        c.scale = scale
        e = np.random.default_rng(seed).uniform(-spread, spread, c.parts[1][1].shape)
        e = np.minimum(e, 7.0)
        c.parts[1][1] = (c.parts[1][1] * 2.0 ** (2 * e)).astype(np.float16)
        c.parts[1][2] = np.clip(-7.5 * c.parts[1][1].astype(np.float64), -65504, 65504).astype(np.float16)
        c.parts[1][1][:, :, ::7] = 0
        want, bound = c.want()
        off = np.abs(f64(c.run(tkdev, c.upload())) - want)
        assert (off <= bound + 2.0**-24 * np.abs(want)).all()


def test_attention_sizes_of_queries_far_apart(torch_cuda, tkdev):
    """Rows of queries of 1e-30, 1 and 1e4, and values in a row from 1e-6 to 1 of its largest."""
    torch = torch_cuda
    c = Case(torch, 12, [60, 61, 62], None, 2, 1, 128, 128, 16, "f32")
    c.q *= torch.tensor([1e-30, 1.0, 1e4], device="cuda")[:, None, None]
    c.q[1] *= torch.logspace(-6, 0, 128, device="cuda")
    want, bound = c.want()
    off = np.abs(f64(c.run(tkdev, c.upload())) - want)
    assert (off <= bound + 2.0**-24 * np.abs(want)).all()


def test_attention_refuses_a_small_workspace(torch_cuda, tkdev):
    c = Case(torch_cuda, 1, [5], None, 1, 1, 64, 64, 16, "f32")
    cache = c.upload()
    c.run(tkdev, cache)
    with pytest.raises(_lib.TKError, match="workspace"):
        ops.kv4_attention(tkdev, cache, c.q, *c.dev_args, c.o, c.ws, c.ws_size - 1, 1, 1, 1, c.width, 1.0)


# ---- a step of them together ---------------------------------------------------------------------

class Server:
    """The buffers of a server's steps: at most `rows` tokens of `batch` requests."""

    def __init__(self, torch, dev, batch, rows, hq, hk, dim, dtype, bs=16, blocks=64, width=12):
        self.torch, self.dev, self.batch, self.rows = torch, dev, batch, rows
        self.hq, self.hk, self.dim, self.dtype, self.bs, self.blocks, self.width = hq, hk, dim, dtype, bs, blocks, width
        self.bufs, self.cache = new_cache(torch, blocks, hk, bs, dim, 64)
        t = kind(torch, dtype)
        self.row = (hq + 2 * hk) * dim
        self.qkv = torch.zeros((rows, self.row), dtype=t, device="cuda")
        self.q = torch.zeros((rows, hq * dim), dtype=t, device="cuda")
        self.k = torch.zeros((rows, hk * dim), dtype=t, device="cuda")
        self.o = torch.full((rows, hq * dim), 3.0, dtype=t, device="cuda")
        turn = torch.outer(torch.arange(width * bs, device="cuda").float(), torch.logspace(0, -3, dim // 2, device="cuda"))
        self.cos, self.sin = turn.cos(), turn.sin()
        self.w = [torch.linspace(0.5, 1.5, dim, device="cuda") for _ in range(2)]
        z = lambda *n: torch.zeros(n, dtype=torch.int32, device="cuda")
        self.ctx, self.new, self.range, self.counts = z(batch), z(batch), z(2), z(4)
        self.free = torch.arange(blocks - 1, -1, -1, dtype=torch.int32, device="cuda")
        self.range[1] = blocks
        self.tables = z(batch, width) - 1
        self.kv, self.start, self.pos, self.slots = z(batch), z(batch + 1), z(rows), z(rows)
        self.ws = torch.empty(ops.kv4_attention_workspace(dev, self.cache, hq), dtype=torch.uint8, device="cuda")

    def step(self, stream):
        v = self.qkv[:, (self.hq + self.hk) * self.dim:]
        ops.paged_slots(self.dev, self.ctx, self.new, self.free, self.range, self.tables, self.kv, self.start, self.pos,
                        self.slots, self.counts, self.batch, self.width, self.bs, self.blocks, self.rows, stream=stream)
        ops.qk_norm_rope(self.dev, self.qkv, self.qkv[:, self.hq * self.dim:], *self.w, self.cos, self.sin, self.pos,
                         self.q, self.k, self.rows, self.hq, self.hk, self.dim, self.dim, self.width * self.bs, 1e-5,
                         self.dtype, q_stride=self.row, k_stride=self.row, stream=stream)
        ops.kv4_append(self.dev, self.cache, self.k, v, self.slots, self.rows, self.dtype, v_stride=self.row, stream=stream)
        ops.kv4_attention(self.dev, self.cache, self.q, self.tables, self.kv, self.start, self.o, self.ws, self.ws.numel(),
                          self.rows, self.batch, self.hq, self.width, self.dim ** -0.5, self.dtype, stream=stream)

    def feed(self, new, seed):
        gen = self.torch.Generator(device="cuda").manual_seed(seed)
        self.qkv.copy_(self.torch.randn(self.qkv.shape, generator=gen, device="cuda"))
        self.new.copy_(i32(self.torch, new))

    def advance(self):
        self.ctx.copy_(self.kv)
        self.range[0] += self.counts[1]


STEPS = [[5, 0, 30], [1, 17, 1], [1, 1, 1], [3, 1, 0], [1, 40, 1]]


@pytest.mark.parametrize("dtype,hq,hk,dim,most", [("f32", 4, 2, 128, 50), ("bf16", 6, 1, 64, 50), ("f16", 2, 2, 256, 50),
                                                  ("bf16", 8, 2, 128, 250), ("f32", 8, 1, 256, 250)])
def test_steps_together_and_captured(torch_cuda, tkdev, dtype, hq, hk, dim, most):
    """Prompts, then single tokens and chunks, of three requests: every step's outputs against the
    oracle over the keys and values of all steps; then the same steps as replays of one captured
    graph (on a stream of its own, with other lengths each time): the same bits."""
    torch = torch_cuda
    plain = Server(torch, tkdev, 3, most, hq, hk, dim, dtype)
    graphed = Server(torch, tkdev, 3, most, hq, hk, dim, dtype)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        graphed.step(side.cuda_stream)
    held = [[np.zeros((0, hk, dim))] * 2 for _ in range(3)]
    for n, new in enumerate(STEPS):
        for s in (plain, graphed):
            s.o.fill_(3.0)
            s.feed(new, n)
        torch.cuda.synchronize()
        plain.step(None)
        tkdev.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        total = sum(new)
        start = np.concatenate([[0], np.cumsum(new)])
        assert plain.start.tolist() == start.tolist() and plain.counts[2] == 0
        assert (plain.o[total:] == 3).all()
        q, k, v = (f64(x[:total]).reshape(total, -1, dim) for x in (plain.q, plain.k, plain.qkv[:, (hq + hk) * dim:]))
        for b in range(3):
            rows = slice(start[b], start[b + 1])
            for i, x in enumerate((k, v)):
                held[b][i] = np.concatenate([held[b][i], oracle4.values_f64(*oracle4.quantise(x[rows], 64))])
            kv = held[b][0].shape[0]
            if new[b] == 0:
                continue
            pad = -kv % 16
            kb, vb = (np.pad(x, ((0, pad), (0, 0), (0, 0))).reshape(-1, 16, hk, dim).transpose(0, 2, 1, 3) for x in held[b])
            want, bound = oracle4.attention_f64(q[rows], kb, vb, 3 * np.abs(kb).max() + 0 * kb, 3 * np.abs(vb).max() + 0 * vb,
                                                np.arange(kb.shape[0])[None], [kv], [0, new[b]], dim ** -0.5, 16)
            y = f64(plain.o[rows]).reshape(want.shape)
            step = HALF_STEP[dtype]
            assert (np.abs(y - want) <= bound + step * np.abs(want) + LEAST[dtype]).all()
            assert np.abs(y - want).max() <= (1e-5 + step) * np.abs(want).max()
        for name in ("o", "tables", "kv", "pos", "slots", "counts"):
            assert torch.equal(getattr(plain, name), getattr(graphed, name)), name
        assert all(torch.equal(a, b) for a, b in zip(plain.bufs, graphed.bufs))
        plain.advance()
        graphed.advance()
    del graph


def test_pages_past_four_gigabytes(torch_cuda, tkdev):
    """The last pages of a cache whose codes have more than 2^32 bytes, and the first of a small one:
    the same keys and values, the same outputs of one token and of a prompt, to the bit."""
    torch = torch_cuda
    hq, hk, dim, ctx, pages = 16, 8, 128, 200, 13
    gen = torch.Generator(device="cuda").manual_seed(91)
    draw = lambda n, h: torch.randn((n, h * dim), generator=gen, device="cuda").half()
    k, v, q = draw(ctx, hk), draw(ctx, hk), draw(100, hq)
    got = []
    for blocks in (pages, 600000):
        assert blocks == pages or blocks * hk * 16 * dim // 2 > 2**32
        codes = [torch.empty((blocks, hk, 16, dim // 2), dtype=torch.uint8, device="cuda") for _ in "kv"]
        pairs = [torch.empty((blocks, hk, 16, 1, 2), dtype=torch.float16, device="cuda") for _ in "kv"]
        cache = ops.kv4_cache(*codes, *pairs, blocks, hk, 16, dim, dim)
        table = torch.arange(blocks - pages, blocks, dtype=torch.int32, device="cuda")
        slots = (table[:, None] * 16 + torch.arange(16, dtype=torch.int32, device="cuda")).flatten()[:ctx].contiguous()
        size = ops.kv4_attention_workspace(tkdev, cache, hq)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        back, one, many = [torch.zeros_like(k) for _ in "kv"], torch.zeros_like(q[:1]), torch.zeros_like(q)
        lens, start = i32(torch, [ctx]), i32(torch, [0, 100])
        torch.cuda.synchronize()
        ops.kv4_append(tkdev, cache, k, v, slots, ctx, "f16")
        ops.kv4_gather(tkdev, cache, slots, *back, ctx, "f16")
        ops.kv4_attention(tkdev, cache, q, table, lens, None, one, ws, size, 1, 1, hq, pages, dim ** -0.5, "f16")
        ops.kv4_attention(tkdev, cache, q, table, lens, start, many, ws, size, 100, 1, hq, pages, dim ** -0.5, "f16")
        got.append(back + [one, many])
        del codes, pairs
    assert all(torch.equal(x, y) for x, y in zip(*got)) and got[0][3].isfinite().all()
    assert (got[0][0] - k).abs().max() < 0.6  # half of a fifteenth of a row's range


def test_two_streams_with_their_own_workspaces(torch_cuda, tkdev):
    """The same cache read from two streams at once, each call with its own workspace and output."""
    torch = torch_cuda
    c = Case(torch, 21, [9000, 500], None, 8, 2, 128, 128, 16, "f32")
    cache = c.upload()
    want = c.run(tkdev, cache).clone()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(c.q) for _ in streams]
    ws = [torch.zeros_like(c.ws) for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, w in zip(streams, outs, ws):
            ops.kv4_attention(tkdev, cache, c.q, *c.dev_args, o, w, c.ws_size, 2, 2, 8, c.width, c.scale, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_prompts_beside_the_gemm_and_captured(torch_cuda, tkdev):
    """Prompts on two streams, one of them a replayed graph, and the INT4 GEMM, which takes all of an
    SM's tensor memory, on a third: the same bits as each alone."""
    torch = torch_cuda
    c = Case(torch, 71, [1500, 700], [130, 64], 8, 4, 128, 128, 16, "bf16", spare=2000)
    cache = c.upload()
    want = c.run(tkdev, cache).clone()
    m, k, n = 64, 1024, 2048
    x = torch.randn(m, k, device="cuda")
    w = torch.randint(0, 256, (k // 2, n), dtype=torch.uint8, device="cuda")
    scales = torch.rand(k // 64, n, device="cuda").half()
    zeros = torch.randint(0, 256, (k // 64, n // 2), dtype=torch.uint8, device="cuda")
    y = torch.zeros(m, n, device="cuda")
    assert ops.path(m, k, n, 64) == 2
    torch.cuda.synchronize()
    ops.qmatmul_int4(tkdev, x, w, scales, zeros, y, m, k, n, 64)
    y0 = y.clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs, ws = [torch.zeros_like(c.q) for _ in "ab"], [torch.zeros_like(c.ws) for _ in "ab"]

    def attend(i, stream):
        ops.kv4_attention(tkdev, cache, c.q, *c.dev_args, outs[i], ws[i], c.ws_size, c.tokens, 2, 8, c.width, c.scale,
                          "bf16", stream=stream.cuda_stream)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        attend(0, streams[0])
        attend(0, streams[0])
    for _ in range(20):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        attend(1, streams[1])
        ops.qmatmul_int4(tkdev, x, w, scales, zeros, y, m, k, n, 64, stream=streams[2].cuda_stream, sync=False)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want) and torch.equal(y, y0)
    tkdev.synchronize()
    del graph


def test_no_tokens_is_no_launch(torch_cuda, tkdev):
    torch = torch_cuda
    c = Case(torch, 1, [5], None, 1, 1, 64, 64, 16, "f32")
    cache = c.upload()
    c.run(tkdev, cache)
    before = tkdev.launch_count()
    ops.kv4_append(tkdev, cache, c.q, c.q, c.dev_args[1], 0)
    ops.kv4_attention(tkdev, cache, c.q, *c.dev_args[:2], c.dev_args[1], c.o, c.ws, c.ws_size, 0, 1, 1, c.width, 1.0)
    assert tkdev.launch_count() == before


def test_kernel_classes(torch_cuda, tkdev):
    """The classes over the framework's own buffers: a prompt, then one token, against the oracle."""
    import tiny_kernel as tk
    hq, hk, dim, bs, width, tokens = 4, 2, 64, 16, 3, 20
    rng = np.random.default_rng(31)
    buf = lambda x, t: tkdev.create_buffer_with_data(t, x)
    new = lambda n, t: tkdev.create_buffer_with_data(t, np.zeros(n))
    slots_of, qk = tk.kernels.kv4.PagedSlots.init(tkdev), tk.kernels.kv4.QKNormRoPE.init(tkdev)
    cache = tk.kernels.kv4.KV4Cache.init(tkdev, 4, hk, bs, dim, 64)
    angles = np.arange(width * bs)[:, None] * 10000.0 ** -(np.arange(dim // 2) / (dim // 2))
    cos, sin = np.cos(angles).astype(np.float32), np.sin(angles).astype(np.float32)
    w = rng.uniform(0.5, 1.5, dim).astype(np.float32)
    tables, free = buf(np.full(width, -1), "i32"), buf([3, 1, 0], "i32")
    held, ctx, taken = [np.zeros((0, hk, dim))] * 2, 0, 0
    for n in (tokens, 1):
        kv, start, pos, slots, counts = (new(m, "i32") for m in (1, 2, n, n, 4))
        slots_of.forward(buf([ctx], "i32"), buf([n], "i32"), free, buf([taken, 3], "i32"), tables, kv, start, pos, slots,
                         counts, bs, 4)
        taken += int(counts.slice()[1])
        assert pos.slice().tolist() == list(range(ctx, ctx + n)) and kv.slice().tolist() == [ctx + n]
        q, k, v = (rng.standard_normal((n, h, dim)).astype(np.float32) for h in (hq, hk, hk))
        qo, ko = new(q.size, "f32"), new(k.size, "f32")
        qk.forward(buf(q, "f32"), buf(k, "f32"), buf(w, "f32"), None, buf(cos, "f32"), buf(sin, "f32"), pos, qo, ko, hq, hk,
                   dim, dim, width * bs, 1e-5)
        qr, kr = qo.slice().reshape(n, hq, dim).copy(), ko.slice().reshape(n, hk, dim).copy()
        norm = np.sqrt((q.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-5)
        y = q / norm * w
        a, b = y[..., :dim // 2], y[..., dim // 2:]
        c, s = (x[ctx:ctx + n, None].astype(np.float64) for x in (cos, sin))
        # at most 64 roundings in the sum of squares (half of it in the root) and 5 more, over sqrt(2) |y|
        atol = 37 * 2.0**-24 * 2**0.5 * np.abs(y).max()
        assert np.allclose(qr, np.concatenate([a * c - b * s, b * c + a * s], -1), rtol=0, atol=atol)
        cache.append(ko, buf(v, "f32"), slots)
        kb, vb = new(k.size, "f32"), new(k.size, "f32")
        cache.gather(slots, kb, vb)
        for i, x in enumerate((kr, v)):
            held[i] = np.concatenate([held[i], oracle4.values_f64(*oracle4.quantise(x, 64))])
        assert np.array_equal(kb.slice().reshape(k.shape), held[0][ctx:].astype(np.float32))
        assert np.array_equal(vb.slice().reshape(v.shape), held[1][ctx:].astype(np.float32))
        o = new(q.size, "f32")
        cache.forward(qo, tables, kv, start, o, hq, dim ** -0.5)
        ctx += n
        pad = -ctx % bs
        kp, vp = (np.pad(x, ((0, pad), (0, 0), (0, 0))).reshape(-1, bs, hk, dim).transpose(0, 2, 1, 3) for x in held)
        want, bound = oracle4.attention_f64(qr.astype(np.float64), kp, vp, 3 * np.abs(kp).max() + 0 * kp,
                                            3 * np.abs(vp).max() + 0 * vp, np.arange(kp.shape[0])[None], [ctx], [0, n],
                                            dim ** -0.5, bs)
        off = np.abs(o.slice().reshape(want.shape) - want)
        assert (off <= bound + 2.0**-24 * np.abs(want) + 2.0**-149).all()
    cache.deinit()
