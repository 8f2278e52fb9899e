"""Every form of the 8-bit product, and every way of it over its tiles, is taken by a shape that the tests run
(test_fp8_forms_gpu.py): by the plan's own word, so that a change of the plan does not leave a form untested."""
import ctypes as C

import pytest

from tiny_kernel import _lib, ops

FORMS = {
    # (m, k, n): (rows, columns, parts of k) of a tile, and whether CTAs walk over several
    # few rows, walking: over blocks of k that end inside a tile's step, over tiles whose last one is ragged
    (5, 300, 40003): (16, 128, 1, True), (16, 640, 40000): (16, 128, 1, True), (20, 1000, 40000): (32, 128, 1, True),
    (40, 640, 40000): (64, 128, 1, True), (64, 1999, 38500): (64, 128, 1, True),
    # few rows, a tile a CTA, and shared by a cluster
    (1, 4096, 14336): (16, 128, 1, False), (3, 2048, 700): (16, 128, 8, False), (30, 14336, 1025): (32, 128, 8, False),
    (60, 4096, 129): (64, 128, 8, False),
    # 128 x 128: alone, shared, walking
    (129, 1100, 129): (128, 128, 1, False), (128, 4096, 4096): (128, 128, 4, False), (250, 2048, 600): (128, 128, 4, False),
    (700, 4096, 1100): (128, 128, 2, False), (20000, 640, 100): (128, 128, 1, True),
    # 128 x 256: a tile a CTA, walking over even and odd numbers of blocks of k
    (777, 640, 5003): (128, 256, 1, False), (777, 2000, 5003): (128, 256, 1, False), (300, 640, 20000): (128, 256, 1, True),
    (513, 1999, 9000): (128, 256, 1, True), (19001, 300, 130): (128, 256, 1, True),
    # pairs of CTAs: a tile each, walking; a last tile of rows that its second CTA has nothing of
    (1500, 8192, 2304): (256, 256, 1, False), (1030, 4096, 5003): (256, 256, 1, True), (640, 4096, 7680): (256, 256, 1, True),
    (257, 4000, 14300): (256, 256, 1, True),
}


@pytest.mark.parametrize("shape", FORMS, ids=lambda s: "x".join(map(str, s)))
def test_the_plan_takes_this_form(shape):
    m, k, n = shape
    rows, cols, parts, at_once = ops.fp8_matmul_plan(m, k, n)
    walks = -(-m // rows) * -(-n // cols) * parts > at_once
    assert (rows, cols, parts, walks) == FORMS[shape]


def test_every_form_is_taken():
    forms = {(rows, cols, parts > 1, walks) for rows, cols, parts, walks in FORMS.values()}
    few = {(rows, 128, *way) for rows in (16, 32, 64) for way in ((True, False), (False, True))} | {(16, 128, False, False)}
    assert forms == few | {(128, 128, False, False), (128, 128, True, False), (128, 128, False, True), (128, 256, False, False),
                           (128, 256, False, True), (256, 256, False, False), (256, 256, False, True)}


def test_plans_cover_their_product():
    """Over the range of sizes: tiles of a known form, parts that each have blocks of k, and no more at once than there are."""
    forms = {(16, 128), (32, 128), (64, 128), (128, 128), (128, 256), (256, 256)}
    for m in (1, 16, 17, 64, 65, 128, 129, 300, 1000, 8192, 2**20):
        for k in (1, 127, 128, 129, 1024, 4100, 16384):
            for n in (1, 100, 129, 2000, 5003, 16384):
                rows, cols, parts, at_once = ops.fp8_matmul_plan(m, k, n)
                tiles = -(-m // rows) * -(-n // cols)
                assert (rows, cols) in forms and parts in (1, 2, 4, 8) and parts <= -(-k // 128)
                assert (rows < 128) == (m <= 64) and (rows > 64 or rows >= m)
                assert 1 <= at_once <= max(296, tiles * parts) and (parts == 1 or at_once == tiles * parts)


def test_refusals():
    L, plan = _lib.lib(), (C.c_uint32 * 4)()
    for args in ((0, 128, 128, 148), (1, 0, 128, 148), (1, 128, 0, 148), (1 << 31, 128, 128, 148), (1, 128, 128, 1),
                 (1, 128, 128, 5000), (1 << 24, 128, 1 << 20, 148)):
        assert L.tk_fp8_matmul_plan(*args, plan) == _lib.TK_ERR_ARG and b"out of range" in L.tk_last_error_string()
    assert L.tk_fp8_matmul_plan(1, 128, 128, 148, None) == _lib.TK_ERR_ARG and b"NULL" in L.tk_last_error_string()
    with pytest.raises(_lib.TKError):
        ops.fp8_matmul_plan(0, 128, 128)
