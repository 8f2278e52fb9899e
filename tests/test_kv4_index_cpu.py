"""The index arithmetic of the 4-bit cache's operators, on the CPU: what the device reads (slots, block
ids, lengths) never becomes an address outside the cache, and 64-bit offsets hold at the largest sizes."""
import ctypes as C
import itertools
import os

import numpy as np
import pytest

import kv4 as oracle4
from tiny_kernel import _lib, ops

INT_MAX, INT_MIN = 2**31 - 1, -2**31
LIB = os.path.join(os.path.dirname(os.path.abspath(oracle4.__file__)), "lib", "libkv4index.so")


@pytest.fixture(scope="module")
def index():
    L = C.CDLL(LIB)  # make -C oracle
    i, n = C.c_int, C.c_longlong
    L.kv4_index_row.argtypes, L.kv4_index_row.restype = [i] * 6, n
    L.kv4_index_slot_row.argtypes, L.kv4_index_slot_row.restype = [i] * 5, n
    L.kv4_index_wanted.argtypes = [i, i]
    L.kv4_index_request.argtypes, L.kv4_index_request.restype = [i, i, n, i, i, i, C.c_void_p], None
    L.kv4_index_tokens_in.argtypes = [i] * 4
    L.kv4_index_new_block.argtypes = [C.c_void_p, i, i, n, i]
    L.kv4_index_prompt_work.argtypes, L.kv4_index_prompt_work.restype = [i] * 5, n
    L.kv4_index_prompt_steps.argtypes = [i] * 6
    L.kv4_index_prompt_find.argtypes = [i] * 5 + [n, C.c_void_p]
    return L


# the last two hold 2^31 - 256 slots, the most that a call takes, at 1 and at 4096 heads
CACHES = [(1, 1, 4), (5, 3, 4), (7, 2, 8), (2**23 - 1, 1, 8), (2**27 - 16, 4096, 4)]


@pytest.mark.parametrize("blocks,heads,shift", CACHES)
def test_rows_of_slots_stay_in_the_cache(index, blocks, heads, shift):
    size = blocks << shift
    inside = sorted({0, 1, (1 << shift) - 1, min(1 << shift, size - 1), size // 2, size - 1})
    for slot, head in itertools.product(inside, sorted({0, heads // 2, heads - 1})):
        want = ((slot >> shift) * heads + head) * (1 << shift) + slot % (1 << shift)
        assert index.kv4_index_slot_row(blocks, heads, shift, slot, head) == want < size * heads
    for slot in (-1, INT_MIN, size, INT_MAX):
        if slot < 0 or slot >= size:
            assert index.kv4_index_slot_row(blocks, heads, shift, slot, 0) == -1
    for block in (-1, INT_MIN, blocks, INT_MAX):
        assert index.kv4_index_row(blocks, heads, shift, block, 0, 0) == -1
    assert index.kv4_index_row(blocks, heads, shift, blocks - 1, heads - 1, (1 << shift) - 1) == size * heads - 1


def test_lengths_at_the_ends_of_their_type(index):
    out = (C.c_int * 4)()
    lens = (INT_MIN, -1, 0, 1, 15, 16, 17, 1000, INT_MAX - 1, INT_MAX)
    for ctx, q, start, shift, width, most in itertools.product(
            lens, lens, (0, 5, 100, 2**40), (4, 8), (1, 3, 2**31 - 9), (1, 100, 2**31 - 9)):
        c = max(ctx, 0)
        want = min(max(q, 0), INT_MAX - c)
        assert index.kv4_index_wanted(ctx, q) == want
        index.kv4_index_request(ctx, q, start, shift, width, most, out)
        n = min(want, max(most - start, 0))
        have = -(-c >> shift)
        need = -(-(c + n) >> shift) if n else have
        assert list(out) == [c, n, min(have, width), min(need, width)]
        # a request's tokens are those of its pages
        if 0 < n <= 1000:
            pages = range(c >> shift, ((c + n - 1) >> shift) + 1)
            assert sum(index.kv4_index_tokens_in(c, n, j, shift) for j in pages) == n
            assert index.kv4_index_tokens_in(c, n, pages[-1] + 1, shift) == 0


def test_pages_off_the_free_list(index):
    ids = np.array([3, -1, 8, 7, 0], np.int32)
    get = lambda begin, end, a, blocks=8: index.kv4_index_new_block(ids.ctypes.data, begin, end, a, blocks)
    assert [get(0, 5, a) for a in range(7)] == [3, -1, -1, 7, 0, -1, -1]  # 8 is none of 8 pages
    assert [get(3, 5, a) for a in range(3)] == [7, 0, -1]
    assert [get(-4, 2, a) for a in range(3)] == [3, -1, -1]  # a negative begin counts as 0
    assert get(5, 0, 0) == get(0, INT_MIN, 0) == get(0, 0, 0) == -1
    assert get(INT_MAX, 5, 2**40) == -1


@pytest.mark.parametrize("per", [1, 2, 3, 5, 128, 200])
def test_work_of_prompts(index, per):
    """A tile's steps cover what its last row sees, by less than two steps; the sums over tiles and the
    search for a step agree with counting one by one."""
    at = C.c_int()
    for n, length, reach, cost in [(1, 1, 999, 1), (1, 0, 999, 1), (200, 50, 999, 1), (300, 300, 2000, 2), (700, 700, 400, 1),
                                   (129, 5000, 9000, 1), (257, 4000, 4096, 1), (640, 100, 999, 1), (1000, 1000, 1024, 1)]:
        last, kv, tiles = length - n, min(length, reach), -(-n * per // 128)
        args = (tiles, per, cost, last, kv)
        steps = [index.kv4_index_prompt_steps(*args, t) for t in range(tiles)]
        for t, s in enumerate(steps):
            sees = min(kv, last + min((t + 1) * 128 - 1, n * per - 1) // per + 1)
            assert -(-max(sees, 0) // 128) <= s - cost <= min(-(-max(sees, 0) // 128) + 1, -(-kv // 128))
        assert index.kv4_index_prompt_work(*args) == sum(steps)
        x = 0
        for t, s in enumerate(steps):
            for j in {0, s // 2, s - 1}:
                assert index.kv4_index_prompt_find(*args, x + j, C.byref(at)) == t and at.value == j
            x += s


def test_work_of_the_largest_prompts(index):
    """2^30 rows, or 2^31 positions: no overflow, and the last step lies in the last tile."""
    at = C.c_int()
    for n, per, kv in [(2**30, 1, 2**31 - 2048), (2**14, 2**16 - 1, 2**31 - 2048), (2**30, 1, 2**30), (1, 2**16 - 1, 1)]:
        tiles = -(-n * per // 128)
        args = (tiles, per, 1, kv - n, kv)
        work, last = index.kv4_index_prompt_work(*args), index.kv4_index_prompt_steps(*args, tiles - 1)
        assert tiles <= work <= tiles * (kv // 128 + 2)
        assert index.kv4_index_prompt_find(*args, work - 1, C.byref(at)) == tiles - 1 and at.value == last - 1
        assert index.kv4_index_prompt_find(*args, 0, C.byref(at)) == 0 and at.value == 0


def test_numpy_numbers_pass_as_arguments():
    """Sizes and factors that are numpy's reach the entry point as the numbers they are."""
    cache = ops.kv4_cache(0x10000, 0x20000, 0x30000, 0x40000, np.int64(8), np.int32(2), 16, 128, 64)
    n = np.int64
    for scale, word in ((np.float32(0.5), "without query_start"), (np.float64("inf"), "scale is not finite")):
        tokens = 3 if word.startswith("without") else 2
        with pytest.raises(_lib.TKError, match=word):
            ops.kv4_attention(0, cache, 0x50000, 0x60000, 0x70000, None, 0x80000, 0x90000, n(10**9), n(tokens), n(2),
                              n(4), n(10), scale)
