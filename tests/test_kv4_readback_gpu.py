"""What the 4-bit cache reads back at the ends of the types."""
import numpy as np
import pytest

import kv4 as oracle4
from test_kv4_gpu import f64, i32, kind, new_cache
from tiny_kernel import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_values_past_the_range_of_f16(torch_cuda, tkdev, dtype):
    """Groups that span f16's range: the scale rounds up, so that the largest value lies past it.  Rounded once to the
    type: an infinity in f16, 65536 in the others."""
    torch = torch_cuda
    x = torch.linspace(-65504, 65504, 64, device="cuda").repeat(2, 1, 1)
    x[1] = x[1].abs() - 65504  # all of it negative: nothing past the range
    x = x.to(kind(torch, dtype))
    x[0, 0, 0], x[0, 0, -1] = -65504, 65504
    bufs, cache = new_cache(torch, 1, 1, 16, 64, 64)
    slots, back = i32(torch, [7, 2]), torch.zeros((2,) + x.shape, dtype=x.dtype, device="cuda")
    torch.cuda.synchronize()
    ops.kv4_append(tkdev, cache, x, x, slots, 2, dtype)
    ops.kv4_gather(tkdev, cache, slots, back[0], back[1], 2, dtype)
    values = oracle4.values_f64(*oracle4.quantise(f64(x), 64))
    assert values.max() == 65536
    want = torch.from_numpy(values).to(x.dtype)
    assert torch.equal(back[0].cpu(), want) and torch.equal(back[1].cpu(), want)
    assert torch.isinf(back[0, 0]).any().item() == (dtype == "f16") and torch.isfinite(back[0, 1]).all()
