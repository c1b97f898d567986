"""Adapters at the limits of their arithmetic, against the formulas in 64 bits."""
import pytest
import torch

from kernelcodegen_amd import ops
from test_gpu_decode_step import DTYPE, generator, ints

pytestmark = pytest.mark.gpu


# ---- add_adapters: h ----

@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("tokens,n,rank", [(1, 200, 16), (70, 328, 16), (40, 100, 40), (40, 100, 128), (30, 70, 256)])
def test_adapters_h_enters_the_second_product_whole(dtype, out, tokens, n, rank):
    """x a is a whole number of 24 binary digits (22 in half precision, times 2^-7) in exact sums; y takes away its first ones, so that what is left
    is exact as well and is rounded once."""
    g = generator(tokens + rank)
    digits, unit = ((65536.0, 256.0, 1.0), 1.0) if dtype == "bf16" else ((2048.0, 1.0), 2.0 ** -7)
    values = [torch.randint(1, 256 if dtype == "bf16" else 2048, (tokens, rank), generator=g, device="cuda").double() * d * unit for d in digits]
    x = torch.stack(values + [torch.zeros_like(values[0])] * (4 - len(digits)), -1).view(tokens, 4 * rank).to(DTYPE[dtype])
    a = torch.eye(rank, device="cuda").repeat_interleave(4, 1)[None].to(DTYPE[dtype])
    j = torch.arange(n, device="cuda") % rank
    b = torch.nn.functional.one_hot(j, rank)[None].to(DTYPE[dtype])
    y = -values[0][:, j].to(DTYPE[out])
    which, scale = ints([0] * tokens), torch.ones(1, device="cuda")
    want = (y.double() + sum(values)[:, j]).to(DTYPE[out])
    assert torch.equal(ops.add_adapters(y, x, a, b, which), want)
    assert torch.equal(ops.add_adapters(y * 0.25, x, a, b, which, scale * 0.25), want * 0.25)
