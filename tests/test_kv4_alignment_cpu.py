"""int32 and f32 arrays off their 4-byte boundary (carved out of a buffer of bytes, say) are refused: a kernel that
read one would fault.  (The arguments are checked before the device, so none is needed.)"""
import pytest

from test_kv4_cpu import A, B, GOOD_ATTENTION, S, T, U, V, W, X, Y, Z, cache, refused
from tiny_kernel import _lib

WORD = "int32 or f32 array is not aligned"


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("n", range(10))
def test_slots(n, off):
    arrays = [A, B, X, Y, Z, W, U, V, S, T]
    arrays[n] += off
    refused(_lib.lib().tk_paged_slots(None, *arrays, 2, 4, 16, 9, 7), WORD)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("n", [2, 3, 4, 5, 6])  # weights, angles, positions
def test_qk(n, off):
    arrays = [U, V, X, Y, A, B, S, Z, W]
    arrays[n] += off
    refused(_lib.lib().tk_qk_norm_rope(None, *arrays, 3, 4, 2, 128, 128, 100, 0, 0, 0, 0, 1e-5, 0, 0), WORD)


@pytest.mark.parametrize("off", [1, 2, 3])
def test_append_and_gather(off):
    L, c = _lib.lib(), cache()
    refused(L.tk_kv4_append(None, c, U, V, S + off, 1, 0, 0, 1), WORD)
    refused(L.tk_kv4_gather(None, c, S + off, U, V, 1, 0, 0, 1), WORD)


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("name", ["tables", "kv_lens", "start"])
def test_attention(name, off):
    a = dict(GOOD_ATTENTION)
    a[name] += off
    refused(_lib.lib().tk_kv4_attention(None, cache(), *a.values()), WORD)
