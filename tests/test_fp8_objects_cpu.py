"""The objects of kernels.fp8 on the CPU: how many rows a call takes, and buffers that do not hold them, which the C call
cannot see.  A call whose buffers hold its rows gets as far as the device, of which there is none."""
import pytest

from tiny_kernel import _lib, ops
from tiny_kernel.kernels import fp8


class Held:
    """A buffer's place and size; nothing reads it."""
    at = 0x10000

    def __init__(self, count):
        self.count = count
        Held.at += 0x1000000
        self.ptr = Held.at


def rows_taken(monkeypatch, call, name):
    seen = {}
    monkeypatch.setattr(ops, name, lambda *a, **k: seen.update(args=a, more=k))
    call()
    return seen


@pytest.mark.parametrize("count,stride,more,rows", [
    (4 * 300, 0, {}, 4), (4 * 300 + 299, 0, {}, 4), (4 * 304, 304, {}, 4), (3 * 304 + 300, 304, {}, 4), (100 * 304, 304, {}, 100),
    (100 * 304, 304, dict(rows=7), 7), (300, 0, dict(rows=1), 1), (299, 0, {}, 0), (0, 304, {}, 0), (5, 0, dict(rows=0), 0)])
def test_rows_of_a_call(monkeypatch, count, stride, more, rows):
    x, scales, codes = Held(300 * max(rows, 1)), Held(3 * max(rows, 1)), Held(count)
    seen = rows_taken(monkeypatch, lambda: fp8.QuantizeFP8.init(0).forward(x, codes, scales, 300, codes_stride=stride, **more),
                      "fp8_quantize")
    assert seen["args"][4:6] == (rows, 300) and seen["more"]["codes_stride"] == (stride or 300)
    seen = rows_taken(monkeypatch, lambda: fp8.AddRMSNormFP8.init(0).forward(
        x, None, None, None, codes, scales, 300, 1e-5, codes_stride=stride, **more), "add_rmsnorm_fp8")
    assert seen["args"][7:9] == (rows, 300) and seen["more"]["codes_stride"] == (stride or 300)


def test_padded_codes_without_their_stride_are_refused():
    """100 rows of 300 in steps of 304 are 101 rows of 300: one more than the other buffers hold."""
    x, codes, scales = Held(100 * 300), Held(100 * 304), Held(100 * 3)
    with pytest.raises(ValueError, match="x holds 30000"):
        fp8.AddRMSNormFP8.init(0).forward(x, None, None, None, codes, scales, 300, 1e-5)
    with pytest.raises(ValueError, match="x holds 30000"):
        fp8.QuantizeFP8.init(0).forward(x, codes, scales, 300)
    with pytest.raises(_lib.TKError, match="device is NULL"):
        fp8.QuantizeFP8.init(0).forward(x, codes, scales, 300, codes_stride=fp8.row(300))


GOOD = dict(x=1200, residual=1200, weight=300, sum_out=1200, codes=3 * 304 + 300, scales=12)


@pytest.mark.parametrize("name", GOOD)
def test_each_buffer_of_the_norm_has_to_hold_its_rows(name):
    def call(sizes):
        fp8.AddRMSNormFP8.init(0).forward(*(Held(v) for v in sizes.values()), 300, 1e-5, rows=4, codes_stride=304)

    with pytest.raises(_lib.TKError, match="device is NULL"):
        call(GOOD)
    with pytest.raises(ValueError, match=name):
        call({**GOOD, name: GOOD[name] - 1})


def test_each_buffer_of_the_product_has_to_hold_its_rows():
    linear = fp8.LinearFP8.__new__(fp8.LinearFP8)
    linear.device, linear.n, linear.k, linear.row = 0, 500, 300, 304
    linear.codes, linear.scales = Held(500 * 304), Held(12)
    good = dict(codes=3 * 304 + 300, scales=12, out=2000)

    def call(sizes):
        linear.forward(*(Held(v) for v in sizes.values()), 4, a_stride=304)

    with pytest.raises(_lib.TKError, match="device is NULL"):
        call(good)
    for name in good:
        with pytest.raises(ValueError, match=name):
            call({**good, name: good[name] - 1})
    with pytest.raises(ValueError, match="weight"):
        linear.load(Held(500 * 300 - 1))


def test_pointers_are_taken_as_they_are():
    with pytest.raises(_lib.TKError, match="device is NULL"):
        fp8.QuantizeFP8.init(0).forward(0x10000, 0x20000, 0x30000, 300, rows=4, codes_stride=304)
