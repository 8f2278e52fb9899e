"""CPU checks of the serving-step operators over the 4-bit cache: every refusal (the arguments are
checked before the device, so none is needed), and the oracle against itself."""
import ctypes as C

import numpy as np
import pytest

import kv4 as oracle4
from tiny_kernel import _lib, ops

A, B, X, Y, Z, W, U, V, S, T = (0x10000 * i for i in range(1, 11))  # addresses; nothing reads them


def refused(status, *words):
    text = _lib.lib().tk_last_error_string().decode()
    assert status == _lib.TK_ERR_ARG, text
    for w in words:
        assert w in text, text


def cache(**over):
    f = dict(k_codes=A, v_codes=B, k_scales=X, v_scales=Y, num_blocks=8, kv_heads=2, block_size=16,
             head_dim=128, group_size=64)
    f.update(over)
    return ops.kv4_cache(**f)


BAD_CACHES = [
    (dict(k_codes=0), "NULL"), (dict(v_scales=0), "NULL"), (dict(v_codes=B + 8), "16-byte"),
    (dict(k_scales=X + 4), "16-byte"), (dict(block_size=8), "block_size 8"),
    (dict(block_size=48), "block_size 48"), (dict(block_size=512), "block_size 512"),
    (dict(head_dim=80), "head_dim 80"), (dict(head_dim=512), "head_dim 512"),
    (dict(group_size=32), "group_size 32"), (dict(head_dim=64, group_size=128), "group_size 128"),
    (dict(num_blocks=0), "out of range"), (dict(kv_heads=0), "out of range"),
    (dict(num_blocks=1 << 27, block_size=16), "out of range"),
]


@pytest.mark.parametrize("over,word", BAD_CACHES)
def test_cache_refusals(over, word):
    L, c = _lib.lib(), cache(**over)
    size = C.c_size_t()
    refused(L.tk_kv4_append(None, c, U, V, S, 1, 0, 0, 0), word)
    refused(L.tk_kv4_gather(None, c, S, U, V, 1, 0, 0, 0), word)
    refused(L.tk_kv4_attention(None, c, U, T, S, None, V, W, 1 << 20, 1, 1, 2, 4, 0, 0, 1.0, 0), word)
    refused(L.tk_kv4_attention_workspace(None, c, 2, C.byref(size)), word)


def test_good_arguments_reach_the_device_check():
    L, c, size = _lib.lib(), cache(), C.c_size_t()
    for st in (L.tk_kv4_append(None, c, U, V, S, 1, 0, 0, 2),
               L.tk_kv4_gather(None, c, S, U, V, 0, 256, 300, 1),
               L.tk_kv4_attention(None, c, U, T, S, None, U, W, 1 << 20, 1, 1, 2, 4, 0, 0, 1.0, 0),
               L.tk_kv4_attention_workspace(None, c, 6, C.byref(size)),
               L.tk_paged_slots(None, A, B, X, Y, Z, W, U, V, S, T, 1, 1, 16, 1, 1),
               L.tk_qk_norm_rope(None, U, V, None, None, A, B, S, U, V, 1, 2, 1, 64, 64, 9, 0, 0, 0,
                                 0, 1e-5, 0, 0),
               L.tk_qk_norm_rope(None, U, None, A, None, None, None, S, U, None, 1, 2, 0, 6, 0, 9, 0,
                                 0, 0, 0, 1e-5, 0, 1)):
        refused(st, "device is NULL")


@pytest.mark.parametrize("args,word", [
    ((0, V, S, 1, 0, 0, 0), "NULL"), ((U, 0, S, 1, 0, 0, 0), "NULL"), ((U, V, 0, 1, 0, 0, 0), "NULL"),
    ((U, V, S, 1, 0, 0, 3), "dtype 3"), ((U, V, S, 1, 0, 0, -1), "dtype -1"),
    ((U, V, S, 1, 255, 0, 0), "k stride 255"), ((U, V, S, 1, 0, 8, 0), "v stride 8"),
    ((U + 2, V, S, 1, 0, 0, 0), "aligned"), ((U, V + 1, S, 1, 0, 0, 1), "aligned"),
    ((U, V, S, 1 << 31, 0, 0, 0), "too many"),
])
def test_append_and_gather_refusals(args, word):
    L, c = _lib.lib(), cache()
    k, v, slots, rest = args[0], args[1], args[2], args[3:]
    refused(L.tk_kv4_append(None, c, k, v, slots, *rest), word)
    refused(L.tk_kv4_gather(None, c, slots, k, v, *rest), word)


def test_gather_refuses_one_buffer_for_both():
    refused(_lib.lib().tk_kv4_gather(None, cache(), S, U, U, 1, 0, 0, 0), "outputs are the same")


GOOD_ATTENTION = dict(q=U, tables=T, kv_lens=S, start=A, o=V, ws=W, size=1 << 30, tokens=3, batch=2,
                      q_heads=4, max_blocks=4, qs=0, os=0, scale=1.0, dtype=0)


@pytest.mark.parametrize("over,word", [
    (dict(q=0), "NULL"), (dict(tables=0), "NULL"), (dict(kv_lens=0), "NULL"), (dict(o=0), "NULL"),
    (dict(ws=0), "NULL"), (dict(ws=W + 8), "16-byte"), (dict(q_heads=3), "q_heads=3"),
    (dict(q_heads=0), "q_heads=0"), (dict(dtype=7), "dtype 7"), (dict(batch=0), "out of range"),
    (dict(max_blocks=0), "out of range"), (dict(tokens=1 << 31), "out of range"),
    (dict(max_blocks=1 << 27), "positions"),
    (dict(start=None), "one token per sequence"), (dict(scale=float("nan")), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(qs=511), "q stride 511"), (dict(os=100), "o stride 100"),
    (dict(o=U, qs=512, os=520), "in place"), (dict(q=U + 2), "aligned"), (dict(o=V + 1, dtype=1), "aligned"),
])
def test_attention_refusals(over, word):
    a = dict(GOOD_ATTENTION, **over)
    refused(_lib.lib().tk_kv4_attention(
        None, cache(), a["q"], a["tables"], a["kv_lens"], a["start"], a["o"], a["ws"], a["size"],
        a["tokens"], a["batch"], a["q_heads"], a["max_blocks"], a["qs"], a["os"], a["scale"],
        a["dtype"]), word)


@pytest.mark.parametrize("over,word", [
    (dict(ctx=0), "NULL"), (dict(counts=0), "NULL"), (dict(kv=A), "output is an input"),
    (dict(counts=Y), "output is an input"), (dict(pos=S), "outputs are the same"),
    (dict(batch=0), "out of range"), (dict(width=0), "out of range"), (dict(blocks=0), "out of range"),
    (dict(tokens=0), "out of range"), (dict(bs=24), "block_size 24"),
    (dict(blocks=1 << 27), "out of range"), (dict(tokens=0x7fffffff), "out of range"),
])
def test_slots_refusals(over, word):
    a = dict(ctx=A, new=B, free=X, rng=Y, tables=Z, kv=W, start=U, pos=V, slots=S, counts=T, batch=2,
             width=4, bs=16, blocks=9, tokens=7)
    a.update(over)
    refused(_lib.lib().tk_paged_slots(None, *a.values()), word)


@pytest.mark.parametrize("over,word", [
    (dict(q=0), "NULL"), (dict(ko=0), "NULL"), (dict(pos=0), "NULL"), (dict(cos=0), "NULL"),
    (dict(d=63), "head_dim=63"), (dict(d=1026), "head_dim=1026"), (dict(d=0), "head_dim=0"),
    (dict(rot=130), "rot_dim=130"), (dict(rot=33), "rot_dim=33"), (dict(hq=0, hk=0), "out of range"),
    (dict(maxp=0), "out of range"), (dict(tokens=0x7fffffff), "out of range"), (dict(dtype=9), "dtype 9"),
    (dict(flags=2), "flags"), (dict(qs=500), "q stride 500"), (dict(kos=200), "k stride 200"),
    (dict(qo=U, qs=600), "in place"), (dict(ko=Z), "outputs are the same"), (dict(q=U + 2), "aligned"),
])
def test_qk_refusals(over, word):
    a = dict(q=U, k=V, wq=None, wk=None, cos=A, sin=B, pos=S, qo=Z, ko=W, tokens=3, hq=4, hk=2, d=128,
             rot=128, maxp=100, qs=0, ks=0, qos=0, kos=0, eps=1e-5, dtype=0, flags=0)
    a.update(over)
    refused(_lib.lib().tk_qk_norm_rope(None, *a.values()), word)


def test_python_refuses_an_unknown_type():
    with pytest.raises(ValueError, match="fp8"):
        ops.kv4_append(0, cache(), U, V, S, 1, "fp8")


def test_oracle_quantisation_covers_the_range():
    x = np.random.default_rng(1).standard_normal((40, 3, 128)) * 3
    codes, s, m = oracle4.quantise(x, 64)
    assert codes.min() == 0 and codes.max() == 15
    assert np.array_equal(oracle4.unpack(oracle4.pack(codes)), codes)
    back = oracle4.values_f64(codes, s, m)
    # half a step, and what the rounding of the offset and of 15 steps adds at the ends of the range
    step = np.repeat(s.astype(np.float64), 64, -1)
    slack = np.abs(np.repeat(m.astype(np.float64), 64, -1)) * 2.0**-11 + 15 * step * 2.0**-11
    assert (np.abs(back - x) <= step / 2 + slack).all()


def test_oracle_attention_of_one_token_is_its_value():
    rng = np.random.default_rng(2)
    k, v = rng.standard_normal((2, 5, 1, 16, 64))
    o, _ = oracle4.attention_f64(rng.standard_normal((1, 3, 64)), k, v, np.abs(k), np.abs(v),
                                 np.array([[3]]), [1], None, 0.125, 16)
    assert np.allclose(o, v[3, 0, 0])


def test_oracle_slots_of_two_requests():
    got = oracle4.paged_slots([5, 0], [12, 2], [7, 4, 9], [0, 3], [[2, -1], [-1, -1]], 16, 10, 16)
    tables, kv, start, pos, slots, counts = got
    assert tables.tolist() == [[2, 7], [4, -1]] and kv.tolist() == [17, 2]
    assert start.tolist() == [0, 12, 14] and pos[:14].tolist() == [*range(5, 17), 0, 1]
    assert slots.tolist() == [*range(37, 48), 112, 64, 65, -1, -1]
    assert counts.tolist() == [14, 2, 0, 2]
