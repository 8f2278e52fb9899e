"""Attention of f32 prompts holds the digits of f32 sums: its error against 64 bits, normwise over all outputs, is
at most 5/4 of that of the same formula in f32 torch operations on the same values (products, exponentials and
sums in f32; the quarter is for the order of torch's own sums, which is not ours to know)."""
import numpy as np
import pytest

from test_kv4_gpu import i32
from tiny_kernel import ops

pytestmark = pytest.mark.gpu


def attention(torch, q, k, v, kv_len, scale, kind):
    """[n, q_heads, dim] of one sequence: q [n, q_heads, dim], k, v [kv_heads, kv_len, dim]."""
    n, hq, dim = q.shape
    per = hq // k.shape[0]
    q = q.to(kind).view(n, -1, per, dim).permute(1, 0, 2, 3).flatten(1, 2)
    score = q @ k.to(kind).transpose(-1, -2) * scale
    sees = kv_len - n + 1 + torch.arange(n, device="cuda").repeat_interleave(per)
    score.masked_fill_(torch.arange(kv_len, device="cuda") >= sees[None, :, None], -torch.inf)
    w = torch.exp(score - score.amax(-1, keepdim=True))
    o = (w @ v.to(kind)) / w.sum(-1, keepdim=True)
    return o.view(-1, n, per, dim).permute(1, 0, 2, 3).flatten(1, 2)


@pytest.mark.parametrize("dim,group,queries", [(64, 64, 256), (128, 64, 256), (128, 128, 256), (256, 64, 100), (256, 128, 100)])
def test_f32_prompts_hold_the_digits_of_f32_sums(torch_cuda, tkdev, dim, group, queries):
    torch = torch_cuda
    hq, hk, bs, lens = 40, 8, 16, [3800, 1700]
    gen = torch.Generator(device="cuda").manual_seed(dim + group)
    pages = [-(-n // bs) for n in lens]
    blocks, width = sum(pages), max(pages)
    tables = np.full((2, width), -1, np.int32)
    tables[0, :pages[0]], tables[1, :pages[1]] = np.arange(pages[0]), pages[0] + np.arange(pages[1])
    bufs, values = [], []
    for _ in "kv":
        codes = torch.randint(0, 16, (blocks, hk, bs, dim), generator=gen, device="cuda", dtype=torch.uint8)
        s = (0.25 * torch.exp(0.4 * torch.randn((blocks, hk, bs, dim // group), generator=gen, device="cuda"))).half()
        m = (-7.5 * s.float() * (1 + 0.1 * torch.randn(s.shape, generator=gen, device="cuda"))).half()
        bufs.append((codes[..., 0::2] | codes[..., 1::2] << 4, torch.stack((s, m), -1)))
        spread = lambda x: x.double().repeat_interleave(group, -1)
        values.append((codes.double() * spread(s) + spread(m)).transpose(0, 1).flatten(1, 2))  # exact
    cache = ops.kv4_cache(bufs[0][0], bufs[1][0], bufs[0][1], bufs[1][1], blocks, hk, bs, dim, group)
    q = torch.randn((2 * queries, hq, dim), generator=gen, device="cuda")
    o = torch.empty_like(q)
    size = ops.kv4_attention_workspace(tkdev, cache, hq)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    args = [i32(torch, x) for x in (tables, lens, [0, queries, 2 * queries])]
    torch.cuda.synchronize()
    ops.kv4_attention(tkdev, cache, q, *args, o, ws, size, 2 * queries, 2, hq, width, dim ** -0.5)
    exact, plain = (torch.cat([attention(torch, q[b * queries:(b + 1) * queries],
                                         *(x[:, first * bs:first * bs + n] for x in values), n, dim ** -0.5, kind).double()
                               for b, (first, n) in enumerate(zip((0, pages[0]), lens))])
                    for kind in (torch.float64, torch.float32))
    off = [float((x.double() - exact).norm() / exact.norm()) for x in (o, plain)]
    assert off[0] <= 1.25 * off[1], off
