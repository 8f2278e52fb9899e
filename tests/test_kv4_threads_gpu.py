"""Calls of the serving step from several threads on one device."""
import ctypes as C
import os

import pytest

import kv4 as oracle4
from test_kv4_gpu import i32, new_cache
from tiny_kernel import _lib

pytestmark = pytest.mark.gpu

LIB = os.path.join(os.path.dirname(os.path.abspath(oracle4.__file__)), "lib", "libthreads.so")  # make -C oracle


def test_launches_of_all_threads_are_counted(torch_cuda, tkdev):
    """Eight native threads, each on its own stream with its own output: every launch is counted once."""
    torch = torch_cuda
    threads, calls = 8, 20000
    bufs, cache = new_cache(torch, 1, 1, 16, 64, 64)
    slots = i32(torch, [3])
    outs = [torch.zeros((2, 64), device="cuda") for _ in range(threads)]
    streams = [torch.cuda.Stream() for _ in range(threads)]
    torch.cuda.synchronize()
    pointers = lambda a: (C.c_void_p * threads)(*a)
    before = tkdev.launch_count()
    failed = C.CDLL(LIB).gather_from_threads(
        C.cast(_lib.lib().tk_kv4_gather_async, C.c_void_p), C.c_void_p(tkdev.handle), C.byref(cache),
        C.c_void_p(slots.data_ptr()), pointers(o[0].data_ptr() for o in outs), pointers(o[1].data_ptr() for o in outs),
        pointers(s.cuda_stream for s in streams), threads, calls)
    torch.cuda.synchronize()
    assert failed == 0
    assert tkdev.launch_count() - before == threads * calls
    assert all((o == 0.25).all() for o in outs)  # codes of 0, scale and offset 0.25
