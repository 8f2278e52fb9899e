"""Kernel wrappers, one module per reference file (src/kernels/*.zig), and beside them kv4: the
serving step over a 4-bit key/value cache; fp8: 8-bit projections; sampler: tokens of a batch."""
from . import fp8, fused, kv4, quantized, rmsnorm, sampler  # noqa: F401
