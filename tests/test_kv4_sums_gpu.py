"""Attention over very long contexts: the sums of numerator and denominator must not drift with their length.

One page is every page of every sequence, so that the tokens' keys and values repeat with the page and the
outputs have a closed form; there are twice as many tiles as CTAs, so that some CTA sums a whole tile.
With weights and scales that repeat, the roundings of a plain running sum go the same way each time: over
131072 positions it is off by 3e-4.
"""
import numpy as np
import pytest

import kv4 as oracle4
from tiny_kernel import ops

pytestmark = pytest.mark.gpu

PAGE = 16


def repeated_page(torch, dev, seed, alike, positions, queries, per, hk, dim, group, scale, tiles, absent=0):
    """(outputs, what they should be, the size of the sums, the size of the scores) of sequences of `positions`
    tokens; alike: the tokens' keys and values are all the same; absent: so many of the first positions have no page."""
    rng = np.random.default_rng(seed)
    shape = (1, hk, PAGE, dim)
    parts = []
    for _ in range(2):
        codes = rng.integers(0, 16, shape).astype(np.uint8)
        s = (0.3 * np.exp(0.5 * rng.standard_normal(shape[:3] + (dim // group,)))).astype(np.float16)
        m = (rng.uniform(-8, 8, s.shape) * s).astype(np.float16)
        if alike:
            for x in (codes, s, m):
                x[:] = x[:, :, :1]
        parts.append((codes, s, m))
    bufs = [torch.from_numpy(oracle4.pack(p[0])).cuda() for p in parts]
    bufs += [torch.from_numpy(np.stack(p[1:], -1)).cuda() for p in parts]
    cache = ops.kv4_cache(*bufs, 1, hk, PAGE, dim, group)
    batch, hq, width = -(-tiles // hk), hk * per, positions // PAGE
    i32 = dict(dtype=torch.int32, device="cuda")
    tables, lens = torch.zeros((batch, width), **i32), torch.full((batch,), positions, **i32)
    tables[:, :absent // PAGE] = -1
    start = torch.arange(0, batch * queries + 1, queries, **i32)
    q1 = rng.standard_normal((queries, hq, dim)).astype(np.float32)
    q = torch.from_numpy(q1).cuda().repeat(batch, 1, 1).contiguous()
    o = torch.full_like(q, 7.0)
    size = ops.kv4_attention_workspace(dev, cache, hq)
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ops.kv4_attention(dev, cache, q, tables, lens, start, o, ws, size, batch * queries, batch, hq, width, scale)
    (kc, ks, km), (vc, vs, vm) = parts
    f64 = lambda x: x.astype(np.float64)
    k, v = oracle4.values_f64(kc, ks, km)[0], oracle4.values_f64(vc, vs, vm)[0]
    # what the products are summed in: 8 * scale + |offset + 8 * scale|, code * scale + |offset|
    centre = np.repeat(8 * f64(vs) + np.abs(f64(vm) + 8 * f64(vs)), group, -1)[0]
    k_size = oracle4.values_f64(kc, ks, np.abs(f64(km)))[0]
    want, sums, most = (np.zeros(q1.shape) for _ in range(3))
    for i in range(queries):
        count = (positions - absent - queries + i + 1 - np.arange(PAGE) + PAGE - 1) // PAGE  # of each token of the page
        for h in range(hq):
            score = scale * (k[h // per] @ f64(q1[i, h]))
            w = count * np.exp(score - score.max())
            w /= w.sum()
            want[i, h], sums[i, h] = w @ v[h // per], w @ centre[h // per]
            most[i, h] = abs(scale) * (k_size[h // per] @ np.abs(f64(q1[i, h]))).max()
    return o.double().cpu().numpy().reshape(batch, queries, hq, dim), want, sums, most


def check(got, want, sums, most, roundings):
    """A weight is off by a factor 1 + eta at most, as in the oracle's bound (scores of f32 sums, the
    exponential); `roundings` are the sums' own, in units of 2^-23 of what they sum."""
    eta = 2 * 2.0**-18 * most + 2.0**-20
    bound = sums * (np.expm1(2 * eta) + roundings * 2.0**-23) + 2.0**-24 * np.abs(want)
    off = np.abs(got - want)
    assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("alike,scale", [(True, 0.0), (False, 0.0), (False, 0.01)])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 128)])
def test_long_prompts(torch_cuda, tkdev, dim, group, alike, scale):
    """64 rows of f32 a tile.  Numerator: the tensor core adds two products for each 16 tokens, each off by 2^-23 of the
    sum at most, for 256 tokens at most: 32.  The offsets' sum and the denominator: 16 to 32 additions in a row
    within a step, 1 of their two halves, 4 of steps, 3 of the parts of a row, each off by half of 2^-23: 20 each.
    Sums of intervals are compensated: 2 more each."""
    ctas = tkdev.sm_count() * (1 if dim == 256 else 2)
    got = repeated_page(torch_cuda, tkdev, dim + group, alike, 131072, 64, 1, 8, dim, group, scale, 2 * ctas)
    check(*got, 32 + 2 * 20 + 3 * 2)


@pytest.mark.parametrize("alike,scale", [(True, 0.0), (False, 0.0), (False, 0.01)])
@pytest.mark.parametrize("queries", [1, 2])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128), (256, 64), (256, 128)])
def test_long_contexts_of_few_rows(torch_cuda, tkdev, dim, group, queries, alike, scale):
    """Four rows (one token) and eight a tile.  Numerator: two products for each 16 tokens of a warp, 512 at
    most before they are set aside: 64.  The offsets' sum and the denominator: 64 additions in a row in a lane,
    5 of lanes, 4 of warps, each off by half of 2^-23: 37 each.  Sums of intervals are compensated: 2 more each."""
    ctas = tkdev.sm_count() * (2 if dim == 256 else 3)
    got = repeated_page(torch_cuda, tkdev, dim + group, alike, 524288, queries, 4, 8, dim, group, scale, 2 * ctas)
    check(*got, 64 + 2 * 37 + 3 * 2)


@pytest.mark.parametrize("rows", ["many", "few"])
@pytest.mark.parametrize("scale,absent", [(3.0, 0), (-3.0, 0), (0.0, 8192), (0.01, 8192), (-3.0, 8192)])
@pytest.mark.parametrize("dim,group", [(64, 64), (128, 64), (128, 128), (256, 128)])
def test_scores_far_from_zero_and_nothing_to_see_at_first(torch_cuda, tkdev, dim, group, scale, absent, rows):
    """Rows whose scores are all far below zero (or above), and rows that have seen nothing when the sums are set
    aside for the first time.  All tokens are alike: whatever the scores, the outputs are the values."""
    queries, per, ctas = (64, 1, 1 if dim == 256 else 2) if rows == "many" else (2, 4, 2 if dim == 256 else 3)
    got, want, sums, _ = repeated_page(torch_cuda, tkdev, dim + group, True, 16384, queries, per, 8, dim, group, scale,
                                       2 * ctas * tkdev.sm_count(), absent)
    check(got, want, sums, np.zeros_like(sums), 64 + 2 * 37 + 3 * 2)
