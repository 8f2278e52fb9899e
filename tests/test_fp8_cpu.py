"""CPU checks of the 8-bit projections and of tk_sample_tokens: every refusal (the arguments are checked
before the device, so none is needed), calls of no rows, and the oracle against itself."""
import numpy as np
import pytest

import fp8
from test_kv4_cpu import A, B, U, V, W, X, Y, Z, refused
from tiny_kernel import _lib, ops

# argument names in the order of the calls; device first
NORM = dict(x=A, residual=B, weight=U, sum_out=X, codes=Y, scales=Z, rows=3, dim=256, x_stride=0, residual_stride=0,
            sum_stride=0, codes_stride=0, eps=1e-5, dtype=0)
QUANTIZE = dict(x=A, codes=Y, scales=Z, rows=3, dim=256, block_rows=1, x_stride=0, codes_stride=0, dtype=1)
MATMUL = dict(a=A, a_scales=B, w=X, w_scales=Y, out=Z, m=3, k=256, n=130, a_stride=0, w_stride=0, out_stride=0, dtype=2)
SAMPLE = dict(logits=A, temperature=B, top_k=U, top_p=V, min_p=W, random=X, tokens=Y, kept=Z, rows=3, vocab=1000,
              stride=0, dtype=0)
CALLS = {"norm": ("tk_add_rmsnorm_fp8", NORM), "quantize": ("tk_fp8_quantize", QUANTIZE),
         "matmul": ("tk_fp8_matmul", MATMUL), "sample": ("tk_sample_tokens", SAMPLE)}


def call(kind, queued=False, **over):
    name, good = CALLS[kind]
    args = [*{**good, **over}.values()]
    L = _lib.lib()
    return getattr(L, name + "_async")(None, *args, None) if queued else getattr(L, name)(None, *args)


REFUSALS = [
    ("norm", dict(x=None), "NULL"), ("norm", dict(codes=None), "NULL"), ("norm", dict(scales=None), "NULL"),
    ("norm", dict(dim=0), "dim=0"), ("norm", dict(dim=32769), "dim=32769"), ("norm", dict(dtype=3), "dtype 3"),
    ("norm", dict(rows=1 << 31), "too many"), ("norm", dict(rows=1 << 30, dim=512), "too many"),
    ("norm", dict(eps=float("nan")), "eps"), ("norm", dict(eps=-1e-5), "eps"), ("norm", dict(eps=float("inf")), "eps"),
    ("norm", dict(x_stride=255), "x stride 255"), ("norm", dict(residual_stride=1), "residual stride"),
    ("norm", dict(sum_stride=8), "sum stride"), ("norm", dict(codes_stride=255), "codes stride"),
    ("norm", dict(x=A + 2), "aligned"), ("norm", dict(residual=B + 1, dtype=2), "aligned"),
    ("norm", dict(sum_out=X + 1, dtype=1), "aligned"), ("norm", dict(weight=U + 2), "aligned"),
    ("norm", dict(scales=Z + 1), "aligned"), ("norm", dict(sum_out=A, x_stride=300), "same stride"),
    ("norm", dict(sum_out=B, sum_stride=300), "same stride"), ("norm", dict(codes=A), "output is an input"),
    ("norm", dict(codes=X), "two outputs"), ("norm", dict(scales=B), "output is an input"),
    ("norm", dict(scales=U), "output is an input"), ("norm", dict(sum_out=U), "output is an input"),
    ("quantize", dict(x=None), "NULL"), ("quantize", dict(codes=None), "NULL"), ("quantize", dict(scales=None), "NULL"),
    ("quantize", dict(block_rows=0), "block_rows=0"), ("quantize", dict(block_rows=64), "block_rows=64"),
    ("quantize", dict(dim=0), "out of range"), ("quantize", dict(rows=1 << 31), "out of range"),
    ("quantize", dict(dim=0x7fffffff), "out of range"), ("quantize", dict(dtype=-1), "dtype -1"),
    ("quantize", dict(x_stride=100), "x stride"), ("quantize", dict(codes_stride=100), "codes stride"),
    ("quantize", dict(x=A + 1), "aligned"), ("quantize", dict(scales=Z + 2), "aligned"),
    ("quantize", dict(codes=A), "output is an input"), ("quantize", dict(scales=Y), "two outputs"),
    ("matmul", dict(a=None), "NULL"), ("matmul", dict(a_scales=None), "NULL"), ("matmul", dict(w=None), "NULL"),
    ("matmul", dict(w_scales=None), "NULL"), ("matmul", dict(out=None), "NULL"), ("matmul", dict(k=0), "out of range"),
    ("matmul", dict(n=0), "out of range"), ("matmul", dict(m=0x7fffffff), "out of range"),
    ("matmul", dict(m=1 << 24, n=1 << 20), "out of range"), ("matmul", dict(k=100), "16-byte"),
    ("matmul", dict(a_stride=264), "16-byte"), ("matmul", dict(w_stride=257), "16-byte"),
    ("matmul", dict(a=A + 8), "16-byte"), ("matmul", dict(w=X + 4), "16-byte"), ("matmul", dict(a_stride=128), "a stride"),
    ("matmul", dict(w_stride=128), "w stride"), ("matmul", dict(out_stride=129), "out stride"),
    ("matmul", dict(out=Z + 1), "aligned"), ("matmul", dict(out=Z + 2, dtype=0), "aligned"),
    ("matmul", dict(a_scales=B + 1), "aligned"), ("matmul", dict(w_scales=Y + 2), "aligned"),
    ("matmul", dict(out=A), "output is an input"), ("matmul", dict(out=Y), "output is an input"),
    ("matmul", dict(dtype=7), "dtype 7"),
    ("sample", dict(logits=None), "NULL"), ("sample", dict(random=None), "NULL"), ("sample", dict(tokens=None), "NULL"),
    ("sample", dict(vocab=0), "out of range"), ("sample", dict(vocab=393217), "out of range"),
    ("sample", dict(rows=(1 << 24) + 1), "out of range"), ("sample", dict(stride=999), "logits stride"),
    ("sample", dict(logits=A + 2), "aligned"), ("sample", dict(logits=A + 1, dtype=1), "aligned"),
    ("sample", dict(top_k=U + 2), "aligned"), ("sample", dict(random=X + 1), "aligned"),
    ("sample", dict(kept=Z + 2), "aligned"), ("sample", dict(tokens=A), "output is an input"),
    ("sample", dict(kept=U), "output is an input"), ("sample", dict(kept=Y), "two outputs"),
    ("sample", dict(dtype=3), "dtype 3"),
]


@pytest.mark.parametrize("kind,over,word", REFUSALS)
def test_refusals(kind, over, word):
    refused(call(kind, **over), word)
    refused(call(kind, queued=True, **over), word)


GOOD = [
    ("norm", {}), ("norm", dict(residual=None, weight=None, sum_out=None)), ("norm", dict(sum_out=A)),
    ("norm", dict(sum_out=B, residual_stride=300, sum_stride=300)), ("norm", dict(dim=1, codes=Y + 1, dtype=2, x=A + 2)),
    ("quantize", {}), ("quantize", dict(block_rows=128, dim=13, codes=Y + 3)), ("matmul", {}),
    ("matmul", dict(k=100, a_stride=112, w_stride=128, out=Z + 2, out_stride=131)), ("sample", {}),
    ("sample", dict(temperature=None, top_k=None, top_p=None, min_p=None, kept=None, vocab=393216)),
]


@pytest.mark.parametrize("kind,over", GOOD)
def test_good_arguments_reach_the_device_check(kind, over):
    refused(call(kind, **over), "device is NULL")


NONE = {"norm": dict(x=None, residual=None, sum_out=None, codes=None, scales=None, rows=0),
        "quantize": dict(x=None, codes=None, scales=None, rows=0),
        "matmul": dict(a=None, a_scales=None, out=None, m=0),
        "sample": dict(logits=None, random=None, tokens=None, kept=None, rows=0)}


@pytest.mark.parametrize("kind", sorted(NONE))
def test_rows_of_no_rows_may_be_null(kind):
    refused(call(kind, **NONE[kind]), "device is NULL")
    rows = "m" if kind == "matmul" else "rows"
    refused(call(kind, **{**NONE[kind], rows: 1}), "NULL argument")


def test_python_calls_pass_their_arguments_on():
    refused_by = []
    for f in (lambda: ops.add_rmsnorm_fp8(0, A, B, U, X, Y, Z, 3, 256, 1e-5, "bf16", x_stride=1),
              lambda: ops.fp8_quantize(0, A, Y, Z, 3, 256, 128, "f16", codes_stride=1),
              lambda: ops.fp8_matmul(0, A, B, X, Y, Z, 3, 256, 130, "f32", out_stride=1),
              lambda: ops.sample_tokens(0, A, None, None, None, None, X, Y, None, 3, 1000, "f16", stride=1)):
        with pytest.raises(_lib.TKError) as e:
            f()
        refused_by.append(str(e.value).split(" stride")[0])
    assert refused_by == ["x", "codes", "out", "logits"]
    with pytest.raises(ValueError):
        ops.fp8_matmul(0, A, B, X, Y, Z, 3, 256, 130, "e4m3")


def test_oracle_codes_are_those_of_the_format():
    import torch
    t = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(t, fp8.TABLE, equal_nan=True) and np.nanmax(fp8.TABLE) == fp8.LARGEST


def test_oracle_sampling_by_hand():
    l = np.log([0.5, 0.1, 0.25, 0.15])
    none = (None, None, None)
    assert [fp8.sample(l, 1, *none, u)[0] for u in (0, 0.49, 0.51, 0.59, 0.61, 0.84, 0.86, 0.999)] == [0, 0, 1, 1, 2, 2, 3, 3]
    assert fp8.sample(l, 1, 2, None, None, 0.7)[:2] == (2, 2)          # 0.5, 0.25
    assert fp8.sample(l, 1, None, 0.6, None, 0.7)[:2] == (2, 2)
    assert fp8.sample(l, 1, None, None, 0.29, 0.99)[:2] == (3, 3)
    assert fp8.sample(l, 1, 3, 0.0, None, 0.99)[:2] == (0, 1)
    assert fp8.sample(l, 0, 3, 0.9, 0.1, 0.99)[:2] == (0, 1)
    assert fp8.sample([1, 3, 3, 3], 1, 2, None, None, 0.6)[:2] == (2, 2)  # equal ones: the lowest indexes
    assert fp8.sample([np.nan, -np.inf], 1, *none, 0.5)[:2] == (-1, 0)
    assert fp8.sample([np.inf, 0, np.inf, np.nan], 1, *none, 0.5)[:2] == (2, 2)
