"""Pointer-level calls into libtkcuda (device pointers as ints, e.g. tensor.data_ptr()).

``stream`` is a CUDA stream handle (int) or None for the device's own stream.  With
``sync=True`` the call is the synchronous entry point (results ready on return, as the
reference's forward() is); otherwise it only enqueues on ``stream``.
"""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import Int4MatrixC, Kv4CacheC, check


_NO_PTR = object()
_tensors = set()  # kinds of objects that have a data_ptr() and no ptr


def _ptr(v) -> int:
    kind = type(v)
    if kind is int or v is None:
        return v
    if kind in _tensors:
        return v.data_ptr()
    ptr = getattr(v, "ptr", _NO_PTR)  # a Buffer's; no error where there is none
    if ptr is not _NO_PTR:
        return ptr
    if not hasattr(v, "data_ptr"):
        return int(v)
    if hasattr(kind, "data_ptr"):
        _tensors.add(kind)
    return v.data_ptr()


def _dev(device) -> int:
    return device.handle if hasattr(device, "handle") else int(device)


def qmatmul_int4(device, x, w_packed, scales, zeros, out, m, k, n, group_size,
                 stream=None, sync=True):
    L = _lib.lib()
    args = (_dev(device), _ptr(x), _ptr(w_packed), _ptr(scales), _ptr(zeros), _ptr(out),
            int(m), int(k), int(n), int(group_size))
    if sync and stream is None:
        check(L.tk_qmatmul_int4(*args))
    else:
        check(L.tk_qmatmul_int4_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def matrix(w_packed, scales, zeros) -> Int4MatrixC:
    return Int4MatrixC(_ptr(w_packed), _ptr(scales), _ptr(zeros))


def int4_ffn(device, x, norm_weight, gate, up, down, out, m, hidden, inter, group_size,
             eps=1e-5, h_out=None, residual=False, stream=None, sync=True, host_io=False):
    """gate/up/down: (w_packed, scales, zeros) triples or Int4MatrixC.  host_io: x and out are
    pinned host buffers (TK_FFN_HOST_IO)."""
    L = _lib.lib()
    mats = [g if isinstance(g, Int4MatrixC) else matrix(*g) for g in (gate, up, down)]
    flags = (_lib.TK_FFN_RESIDUAL if residual else 0) | (_lib.TK_FFN_HOST_IO if host_io else 0)
    args = (_dev(device), _ptr(x), _ptr(norm_weight), C.byref(mats[0]), C.byref(mats[1]),
            C.byref(mats[2]), _ptr(out), _ptr(h_out), int(m), int(hidden), int(inter),
            int(group_size), float(eps), flags)
    if sync and stream is None:
        check(L.tk_int4_ffn(*args))
    else:
        check(L.tk_int4_ffn_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def rmsnorm(device, x, weight, out, rows, dim, eps, stream=None, sync=True):
    L = _lib.lib()
    args = (_dev(device), _ptr(x), _ptr(weight), _ptr(out), int(rows), int(dim), float(eps))
    if sync and stream is None:
        check(L.tk_rmsnorm(*args))
    else:
        check(L.tk_rmsnorm_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def fused_rmsnorm_rope(device, x, weight, cos_cache, sin_cache, out, rows, dim, head_dim, pos,
                       eps, stream=None, sync=True):
    L = _lib.lib()
    args = (_dev(device), _ptr(x), _ptr(weight), _ptr(cos_cache), _ptr(sin_cache), _ptr(out),
            int(rows), int(dim), int(head_dim), int(pos), float(eps))
    if sync and stream is None:
        check(L.tk_fused_rmsnorm_rope(*args))
    else:
        check(L.tk_fused_rmsnorm_rope_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def silu_mul(device, gate, up, out, n, stream=None, sync=True):
    L = _lib.lib()
    args = (_dev(device), _ptr(gate), _ptr(up), _ptr(out), int(n))
    if sync and stream is None:
        check(L.tk_silu_mul(*args))
    else:
        check(L.tk_silu_mul_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def matvec(device, x, W, out, K, N, stream=None, sync=True):
    """out[n] = sum_k W[n][k] x[k], W f32 [N][K] (Matvec, fused.zig:53-89)."""
    L = _lib.lib()
    args = (_dev(device), _ptr(x), _ptr(W), _ptr(out), int(K), int(N))
    if sync and stream is None:
        check(L.tk_matvec(*args))
    else:
        check(L.tk_matvec_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def matvec_dual(device, x, W1, W2, out1, out2, K, N, stream=None, sync=True):
    """Two matvecs sharing x (MatvecDual, fused.zig:91-133)."""
    L = _lib.lib()
    args = (_dev(device), _ptr(x), _ptr(W1), _ptr(W2), _ptr(out1), _ptr(out2), int(K), int(N))
    if sync and stream is None:
        check(L.tk_matvec_dual(*args))
    else:
        check(L.tk_matvec_dual_async(*args, stream))
        if sync:
            check(L.tk_device_synchronize(_dev(device)))


def repack_q4_0(device, blocks, w_packed, scales, zeros, n_rows, k, order=0):
    """GGUF Q4_0 blocks [n_rows][k/32] x 18 B -> qmatmul_int4 layout, group size 32
    (order 0: the reference loader's nibble order, 1: ggml's)."""
    check(_lib.lib().tk_repack_q4_0(_dev(device), _ptr(blocks), _ptr(w_packed), _ptr(scales),
                                    _ptr(zeros), int(n_rows), int(k), int(order)))


def paged_attention(device, q, k_cache, v_cache, block_tables, context_lens, o, batch,
                    num_heads, head_dim, max_blocks):
    """PagedAttention.forward (attention.zig:51-100): decode attention over block-tabled caches."""
    check(_lib.lib().tk_paged_attention(_dev(device), _ptr(q), _ptr(k_cache), _ptr(v_cache),
                                        _ptr(block_tables), _ptr(context_lens), _ptr(o),
                                        int(batch), int(num_heads), int(head_dim),
                                        int(max_blocks)))


_TYPES = {"f32": _lib.TK_F32, "f16": _lib.TK_F16, "bf16": _lib.TK_BF16}


def _dtype(dtype) -> int:
    """A TK_* type code from "f32", "f16", "bf16" or the code itself."""
    if isinstance(dtype, str):
        if dtype not in _TYPES:
            raise ValueError(f"unknown dtype {dtype!r}: f32, f16 or bf16")
        return _TYPES[dtype]
    return int(dtype)


_entries = {}  # name -> (synchronous entry point, queued one)


def _number(v):
    """An argument that ctypes did not take as it was: other kinds of numbers (numpy's)."""
    if v is None or isinstance(v, (int, float)) or not hasattr(v, "__float__"):
        return v
    return int(v) if hasattr(v, "__index__") else float(v)


def _call(name, args, stream, sync):
    """The synchronous entry point, or with a stream (or sync=False) the one that only queues."""
    entry = _entries.get(name)
    if entry is None:
        L = _lib.lib()
        entry = _entries[name] = (getattr(L, name), getattr(L, name + "_async"))
    if stream is None and sync:
        fn = entry[0]
    else:
        fn = entry[1]
        args += (stream,)
    try:
        status = fn(*args)
    except C.ArgumentError:
        status = fn(*map(_number, args))
    if status:
        check(status)


def paged_slots(device, context_lens, query_lens, free_blocks, free_range, block_tables, kv_lens,
                query_start, positions, slots, counts, batch, max_blocks, block_size, num_blocks,
                max_tokens, stream=None, sync=True):
    """Block tables, positions and slots of a step from the requests' lengths (int32 buffers)."""
    _call("tk_paged_slots",
          (_dev(device), _ptr(context_lens), _ptr(query_lens), _ptr(free_blocks), _ptr(free_range),
           _ptr(block_tables), _ptr(kv_lens), _ptr(query_start), _ptr(positions), _ptr(slots),
           _ptr(counts), batch, max_blocks, block_size, num_blocks,
           max_tokens), stream, sync)


def qk_norm_rope(device, q, k, q_weight, k_weight, cos_cache, sin_cache, positions, q_out, k_out,
                 tokens, q_heads, kv_heads, head_dim, rot_dim, max_pos, eps, dtype="f32",
                 interleaved=False, q_stride=0, k_stride=0, q_out_stride=0, k_out_stride=0,
                 stream=None, sync=True):
    """Per-head norm (a None weight: none) and rotation of queries and keys at their positions."""
    _call("tk_qk_norm_rope",
          (_dev(device), _ptr(q), _ptr(k), _ptr(q_weight), _ptr(k_weight), _ptr(cos_cache),
           _ptr(sin_cache), _ptr(positions), _ptr(q_out), _ptr(k_out), tokens, q_heads,
           kv_heads, head_dim, rot_dim, max_pos, q_stride, k_stride,
           q_out_stride, k_out_stride, eps, _dtype(dtype),
           _lib.TK_ROPE_INTERLEAVED if interleaved else 0), stream, sync)


def kv4_cache(k_codes, v_codes, k_scales, v_scales, num_blocks, kv_heads, block_size, head_dim,
              group_size) -> Kv4CacheC:
    """The description of a 4-bit cache that the kv4_* calls take (the buffers stay the caller's)."""
    return Kv4CacheC(_ptr(k_codes), _ptr(v_codes), _ptr(k_scales), _ptr(v_scales), int(num_blocks),
                     int(kv_heads), int(block_size), int(head_dim), int(group_size))


def kv4_append(device, cache, k, v, slots, tokens, dtype="f32", k_stride=0, v_stride=0, stream=None,
               sync=True):
    """Keys and values quantised into their slots (-1: not written)."""
    _call("tk_kv4_append",
          (_dev(device), C.byref(cache), _ptr(k), _ptr(v), _ptr(slots), tokens, k_stride,
           v_stride, _dtype(dtype)), stream, sync)


def kv4_gather(device, cache, slots, k, v, tokens, dtype="f32", k_stride=0, v_stride=0, stream=None,
               sync=True):
    """Keys and values of slots read back from the cache (-1: the row stays)."""
    _call("tk_kv4_gather",
          (_dev(device), C.byref(cache), _ptr(slots), _ptr(k), _ptr(v), tokens, k_stride,
           v_stride, _dtype(dtype)), stream, sync)


def kv4_attention_workspace(device, cache, q_heads) -> int:
    """Bytes of the workspace that kv4_attention needs."""
    size = C.c_size_t()
    check(_lib.lib().tk_kv4_attention_workspace(_dev(device), C.byref(cache), int(q_heads),
                                                C.byref(size)))
    return size.value


def kv4_attention(device, cache, q, block_tables, kv_lens, query_start, o, workspace,
                  workspace_bytes, tokens, batch, q_heads, max_blocks, scale, dtype="f32",
                  q_stride=0, o_stride=0, stream=None, sync=True):
    """Attention of the step's queries over the 4-bit pages (query_start None: one token each)."""
    _call("tk_kv4_attention",
          (_dev(device), C.byref(cache), _ptr(q), _ptr(block_tables), _ptr(kv_lens),
           _ptr(query_start), _ptr(o), _ptr(workspace), workspace_bytes, tokens,
           batch, q_heads, max_blocks, q_stride, o_stride, scale,
           _dtype(dtype)), stream, sync)


def argmax(device, x, n, out):
    """out[0] = index of the largest of x[0..n) (ties: the smallest index)."""
    check(_lib.lib().tk_argmax(_dev(device), _ptr(x), int(n), _ptr(out)))


def softmax_sample(device, logits, probs, sampled, vocab, temperature, random_val):
    """probs = softmax(logits / temperature); sampled[0] = first index whose cumulative
    probability exceeds random_val (shaders.zig:826-887)."""
    check(_lib.lib().tk_softmax_sample(_dev(device), _ptr(logits), _ptr(probs), _ptr(sampled),
                                       int(vocab), float(temperature), float(random_val)))


def dequant_int4(device, w_packed, scales, zeros, out, k, n, group_size):
    check(_lib.lib().tk_dequant_int4(_dev(device), _ptr(w_packed), _ptr(scales), _ptr(zeros),
                                     _ptr(out), int(k), int(n), int(group_size)))


def path(m, k, n, group_size) -> int:
    """qmatmul_int4's path: 3 = batch 1-2 decode kernel, 2 = tcgen05 GEMM, 1 = streaming engine,
    0 = CUDA-core fallback, -1 = invalid shape."""
    return _lib.lib().tk_qmatmul_int4_path(int(m), int(k), int(n), int(group_size))


def ffn_path(m, hidden, inter, group_size) -> int:
    """int4_ffn's path, with the same codes as path()."""
    return _lib.lib().tk_int4_ffn_path(int(m), int(hidden), int(inter), int(group_size))
