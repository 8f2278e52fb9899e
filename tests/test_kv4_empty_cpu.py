"""A call of the serving step with no tokens: the rows' pointers may be NULL, as those of empty tensors are; all
other arguments are checked as ever.  (The arguments are checked before the device, so none is needed.)"""
import pytest

from test_kv4_cpu import A, B, S, T, U, V, W, cache, refused
from tiny_kernel import _lib

NULL = None


def calls(tokens, row):
    """Each call with `tokens` tokens and `row` in the place of every pointer to rows."""
    L, c = _lib.lib(), cache()
    return {
        "append": lambda: L.tk_kv4_append(None, c, row, row, row, tokens, 0, 0, 0),
        "gather": lambda: L.tk_kv4_gather(None, c, row, row, row, tokens, 0, 0, 0),
        "qk": lambda: L.tk_qk_norm_rope(None, row, row, A, B, U, V, row, row, row, tokens, 4, 2, 128, 128, 9, 0, 800, 0, 0,
                                        1e-5, 0, 0),
        "attention": lambda: L.tk_kv4_attention(None, c, row, T, S, A, row, W, 1 << 30, tokens, 2, 4, 4, 0, 600, 1.0, 0),
    }


@pytest.mark.parametrize("name", ["append", "gather", "qk", "attention"])
def test_rows_of_no_tokens_may_be_null(name):
    refused(calls(0, NULL)[name](), "device is NULL")
    refused(calls(1, NULL)[name](), "NULL argument")


def test_other_arguments_of_no_tokens_are_checked():
    L = _lib.lib()
    refused(L.tk_kv4_append(None, cache(head_dim=80), NULL, NULL, NULL, 0, 0, 0, 0), "head_dim 80")
    refused(L.tk_kv4_gather(None, cache(), NULL, NULL, NULL, 0, 0, 0, 5), "dtype 5")
    refused(L.tk_qk_norm_rope(None, NULL, NULL, A, B, NULL, V, NULL, NULL, NULL, 0, 4, 2, 128, 128, 9, 0, 0, 0, 0, 1e-5, 0, 0),
            "NULL argument")
    refused(L.tk_kv4_attention(None, cache(), NULL, T, NULL, A, NULL, W, 1 << 30, 0, 2, 4, 4, 0, 0, 1.0, 0), "NULL argument")
    refused(L.tk_kv4_attention(None, cache(), NULL, T, S, A, NULL, W, 1 << 30, 0, 2, 3, 4, 0, 0, 1.0, 0), "q_heads=3")
