"""Projections in 8-bit floating point and the norm before them (no file of the reference; next to its
RMSNorm, src/kernels/rmsnorm.zig:6-43, and QMatMulInt4, src/kernels/quantized.zig:6-51).  Every
forward() is synchronous; streams and graphs go through the functions of ops."""
from __future__ import annotations

from .. import _lib, ops

BLOCK = 128


def blocks(n: int) -> int:
    """Blocks of 128 that n values make."""
    return -(-int(n) // BLOCK)


def row(k: int) -> int:
    """Bytes from one row of k codes to the next that the product takes: on 16-byte boundaries."""
    return -(-int(k) // 16) * 16


def _span(rows: int, stride: int, dim: int) -> int:
    """Elements from the first to the last of rows of dim values, stride apart."""
    return (rows - 1) * stride + dim if rows else 0


def _rows_of(codes, rows, stride: int, dim: int) -> int:
    """rows, or (None) as many as codes hold."""
    return int(rows) if rows is not None else max(0, codes.count - dim + stride) // stride


def _check(**needs) -> None:
    """name=(buffer, elements that the call reads or writes of it); pointers and tensors are not known."""
    for name, (buffer, elements) in needs.items():
        count = getattr(buffer, "count", None)
        if isinstance(count, int) and count < elements:
            raise ValueError(f"{name} holds {count} elements of {elements}")


class AddRMSNormFP8:
    """x + residual (None: x alone), its RMS norm as e4m3 codes [rows][dim] (u8) and scales
    [rows][blocks(dim)] (f32), and the sum itself (a None sum_out: not written).  Rows of codes lie
    codes_stride bytes apart (0: dim; LinearFP8 takes its own .row); rows None: as many as codes hold."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "AddRMSNormFP8":
        return cls(device)

    def forward(self, x, residual, weight, sum_out, codes, scales, dim, eps, dtype="f32", rows=None,
                codes_stride=0):
        dim, stride = int(dim), int(codes_stride) or int(dim)
        rows = _rows_of(codes, rows, stride, dim)
        _check(x=(x, rows * dim), residual=(residual, rows * dim), weight=(weight, dim),
               sum_out=(sum_out, rows * dim), codes=(codes, _span(rows, stride, dim)),
               scales=(scales, rows * blocks(dim)))
        ops.add_rmsnorm_fp8(self.device, x, residual, weight, sum_out, codes, scales, rows, dim, eps, dtype,
                            codes_stride=stride)


class QuantizeFP8:
    """Codes and scales of activations that no norm precedes; rows and codes_stride as above."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "QuantizeFP8":
        return cls(device)

    def forward(self, x, codes, scales, dim, dtype="f32", rows=None, codes_stride=0):
        dim, stride = int(dim), int(codes_stride) or int(dim)
        rows = _rows_of(codes, rows, stride, dim)
        _check(x=(x, rows * dim), codes=(codes, _span(rows, stride, dim)), scales=(scales, rows * blocks(dim)))
        ops.fp8_quantize(self.device, x, codes, scales, rows, dim, 1, dtype, codes_stride=stride)


class LinearFP8:
    """A weight [n][k] (out_dim, in_dim) in blocks of 128 x 128 that owns its buffers (device memory; rows
    of codes on 16-byte boundaries), and the product with it."""

    def __init__(self, device, n, k):
        self.device, self.n, self.k = device, int(n), int(k)
        self.row = row(k)
        self.codes = device.create_buffer("u8", self.n * self.row, _lib.TK_MEM_DEVICE)
        self.scales = device.create_buffer("f32", blocks(n) * blocks(k), _lib.TK_MEM_DEVICE)

    @classmethod
    def init(cls, device, n, k) -> "LinearFP8":
        return cls(device, n, k)

    def load(self, weight, dtype="f32"):
        """Quantises weight, n rows of k values of type dtype."""
        _check(weight=(weight, self.n * self.k))
        ops.fp8_quantize(self.device, weight, self.codes, self.scales, self.n, self.k, BLOCK, dtype,
                         codes_stride=self.row)

    def forward(self, codes, scales, out, m, dtype="f32", a_stride=0):
        """out [m][n] of m rows of activations (a_stride bytes apart, 0: k)."""
        m, stride = int(m), int(a_stride) or self.k
        _check(codes=(codes, _span(m, stride, self.k)), scales=(scales, m * blocks(self.k)), out=(out, m * self.n))
        ops.fp8_matmul(self.device, codes, scales, self.codes, self.scales, out, m, self.k, self.n,
                       dtype, a_stride=stride, w_stride=self.row)

    def deinit(self) -> None:
        for b in (self.codes, self.scales):
            b.deinit()
