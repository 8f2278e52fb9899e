"""Norm and rotation into rows apart from each other, of another distance than the inputs'."""
import pytest

from test_kv4_gpu import check_qk, qk_case
from tiny_kernel import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,rot,inter,gap,at", [(128, 128, False, 24, 8), (128, 64, True, 3, 1), (64, 32, False, 8, 0),
                                                  (6, 2, False, 5, 2), (256, 256, False, 4, 4)])
def test_strided_outputs(torch_cuda, tkdev, dim, rot, inter, gap, at, dtype):
    """Queries and keys into one row of outputs with a gap before, between and behind them, which stays as it was."""
    torch = torch_cuda
    tokens, hq, hk = 9, 5, 2
    x, w, cos, sin, pos, far, row = qk_case(torch, dim + gap, tokens, hq, hk, dim, rot, True, dtype, 0, 0)
    wide = at + hq * dim + gap + hk * dim + gap
    out = torch.full((tokens, wide), 7.0, dtype=x.dtype, device="cuda")
    qo, ko = out[:, at:], out[:, at + hq * dim + gap:]
    torch.cuda.synchronize()
    ops.qk_norm_rope(tkdev, x, x[:, hq * dim:], *w, cos, sin, pos, qo, ko, tokens, hq, hk, dim, rot, far, 1e-5, dtype,
                     interleaved=inter, q_stride=row, k_stride=row, q_out_stride=wide, k_out_stride=wide)
    for y, first, m, wt in ((qo, 0, hq, w[0]), (ko, hq * dim, hk, w[1])):
        check_qk(y[:, :m * dim].unflatten(1, (m, dim)), x[:, first:first + m * dim].unflatten(1, (m, dim)), wt, cos, sin, pos,
                 rot, inter, dtype)
        y[:, :m * dim] = 7
    assert (out == 7).all()
