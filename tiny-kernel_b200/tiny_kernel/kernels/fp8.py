"""Projections in 8-bit floating point and the norm before them (no file of the reference; next to its
RMSNorm, src/kernels/rmsnorm.zig:6-43, and QMatMulInt4, src/kernels/quantized.zig:6-51).  Every
forward() is synchronous; streams and graphs go through the functions of ops."""
from __future__ import annotations

from .. import _lib, ops

BLOCK = 128


def blocks(n: int) -> int:
    """Blocks of 128 that n values make."""
    return -(-int(n) // BLOCK)


class AddRMSNormFP8:
    """x + residual (None: x alone), its RMS norm as e4m3 codes [rows][dim] (u8) and scales
    [rows][blocks(dim)] (f32), and the sum itself (a None sum_out: not written)."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "AddRMSNormFP8":
        return cls(device)

    def forward(self, x, residual, weight, sum_out, codes, scales, dim, eps, dtype="f32"):
        ops.add_rmsnorm_fp8(self.device, x, residual, weight, sum_out, codes, scales,
                            codes.count // int(dim), dim, eps, dtype)


class QuantizeFP8:
    """Codes and scales of activations that no norm precedes."""

    def __init__(self, device):
        self.device = device

    @classmethod
    def init(cls, device) -> "QuantizeFP8":
        return cls(device)

    def forward(self, x, codes, scales, dim, dtype="f32"):
        ops.fp8_quantize(self.device, x, codes, scales, codes.count // int(dim), dim, 1, dtype)


class LinearFP8:
    """A weight [n][k] (out_dim, in_dim) in blocks of 128 x 128 that owns its buffers (device memory; rows
    of codes on 16-byte boundaries), and the product with it."""

    def __init__(self, device, n, k):
        self.device, self.n, self.k = device, int(n), int(k)
        self.row = -(-self.k // 16) * 16
        self.codes = device.create_buffer("u8", self.n * self.row, _lib.TK_MEM_DEVICE)
        self.scales = device.create_buffer("f32", blocks(n) * blocks(k), _lib.TK_MEM_DEVICE)

    @classmethod
    def init(cls, device, n, k) -> "LinearFP8":
        return cls(device, n, k)

    def load(self, weight, dtype="f32"):
        """Quantises weight, n rows of k values of type dtype."""
        ops.fp8_quantize(self.device, weight, self.codes, self.scales, self.n, self.k, BLOCK, dtype,
                         codes_stride=self.row)

    def forward(self, codes, scales, out, m, dtype="f32", a_stride=0):
        """out [m][n] of m rows of activations (a_stride bytes apart, 0: k)."""
        ops.fp8_matmul(self.device, codes, scales, self.codes, self.scales, out, m, self.k, self.n,
                       dtype, a_stride=a_stride, w_stride=self.row)

    def deinit(self) -> None:
        for b in (self.codes, self.scales):
            b.deinit()
