"""The objects of kernels.fp8 one after the other on the device, at a width whose rows of codes the product wants padded."""
import numpy as np
import pytest

import fp8
from test_fp8_gpu import NORM_ERROR, check_codes
from tiny_kernel import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,k,n", [(4, 300, 500), (100, 300, 70), (1, 17, 130), (90, 1000, 64), (5, 256, 300)])
def test_norm_and_quantisation_feed_the_product(torch_cuda, tkdev, m, k, n):
    rng = np.random.default_rng(m + k)
    x, r, weight = rng.normal(size=(m, k)), rng.normal(size=(m, k)), 1 + 0.1 * rng.normal(size=k)
    buf = lambda a: tkdev.create_buffer_with_data("f32", np.asarray(a, np.float32))
    new = lambda t, c: tkdev.create_buffer_with_data(t, np.full(c, 7))
    objects = kernels.fp8
    linear = objects.LinearFP8.init(tkdev, n, k)
    linear.load(buf(rng.normal(size=(n, k)) * k**-0.5))
    assert linear.row == objects.row(k)
    w = linear.codes.read().reshape(n, -1)[:, :k], linear.scales.read().reshape(objects.blocks(n), -1)
    total = new("f32", m * k)
    for norm in (True, False):
        codes, scales, y = new("u8", m * linear.row), new("f32", m * objects.blocks(k)), new("f32", m * n)
        if norm:
            objects.AddRMSNormFP8.init(tkdev).forward(buf(x), buf(r), buf(weight), total, codes, scales, k, 1e-5,
                                                      codes_stride=linear.row)
            _, values = fp8.add_rmsnorm(x.astype(np.float32), r.astype(np.float32), weight.astype(np.float32), 1e-5)
        else:
            objects.QuantizeFP8.init(tkdev).forward(total, codes, scales, k, rows=m, codes_stride=linear.row)
            values = total.read().reshape(m, k).astype(np.float64)
        a, a_scales = codes.read().reshape(m, -1), scales.read().reshape(m, -1)
        check_codes(values, a[:, :k], a_scales.astype(np.float64), fp8.group_scales(values, 1), 1, NORM_ERROR if norm else 0)
        assert (a[:, k:] == 7).all()
        linear.forward(codes, scales, y, m, a_stride=linear.row)
        want, size = fp8.matmul(a[:, :k], a_scales, *w)
        assert (np.abs(y.read().reshape(m, n) - want) <= 140 * 2.0**-23 * size).all()
    linear.deinit()
