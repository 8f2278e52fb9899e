"""Kernel wrappers, one module per reference file (src/kernels/*.zig), and kv4: the serving step
over a 4-bit key/value cache."""
from . import fused, kv4, quantized, rmsnorm  # noqa: F401
