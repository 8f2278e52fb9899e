"""Steps without tokens over empty tensors."""
import pytest

from test_kv4_gpu import Case
from tiny_kernel import ops

pytestmark = pytest.mark.gpu


def test_empty_tensors(torch_cuda, tkdev):
    torch = torch_cuda
    c = Case(torch, 1, [5], None, 2, 1, 64, 64, 16, "f32")
    cache = c.upload()
    c.run(tkdev, cache)
    before, launches = [b.clone() for b in c.bufs], tkdev.launch_count()
    rows, which = torch.empty((0, 128), device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda")
    turn = torch.ones((9, 32), device="cuda")
    ops.qk_norm_rope(tkdev, rows, rows, None, None, turn, turn, which, rows, rows, 0, 2, 1, 64, 64, 9, 1e-5)
    ops.kv4_append(tkdev, cache, rows, rows, which, 0)
    ops.kv4_gather(tkdev, cache, which, rows, rows, 0)
    start = torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.kv4_attention(tkdev, cache, rows, *c.dev_args[:2], start, rows, c.ws, c.ws_size, 0, 1, 2, c.width, 1.0)
    tkdev.synchronize()
    assert tkdev.launch_count() == launches and all(torch.equal(a, b) for a, b in zip(c.bufs, before))
