"""Adapters at the limits of their arithmetic, against the formulas in 64 bits."""
import pytest
import torch

from kernelcodegen_amd import ops
from test_gpu_answer_operators import adapters_case, check_adapters
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


# ---- add_adapters: more than 1024 tokens ----

@pytest.mark.parametrize("dtype,out,tokens,n,k,rank,runs", [
    ("bf16", "bf16", 1025, 1280, 264, 8, False), ("f16", "f32", 1025, 1280, 264, 16, False), ("bf16", "f32", 2600, 6400, 1032, 8, True), ("bf16", "bf16", 2600, 1003, 2048, 64, True),
    ("f16", "f16", 1300, 1280, 520, 64, False), ("bf16", "bf16", 1100, 1024, 520, 128, True), ("f16", "f32", 1100, 1003, 520, 128, False), ("bf16", "f32", 1025, 640, 264, 256, False),
    ("f16", "f16", 1100, 1024, 264, 24, True)])
def test_adapters_of_more_than_a_thousand_tokens(dtype, out, tokens, n, k, rank, runs):
    """The forms that the rule takes for prompts: other tiles, parts of k by the rank, one pass over the columns and (6400 of fp32) several; columns that are a whole
    number of a workgroup's and others; runs of one adapter, and several in each tile."""
    y, x, a, b, which, scale = adapters_case(tokens + rank, tokens, n, k, rank, 7, dtype, out)
    if runs:
        which = which.sort().values.contiguous()
    got = ops.add_adapters(y, x, a, b, which, scale)
    for at in (slice(None, 70), slice(tokens // 2 - 9, None, 29), slice(-40, None)):
        check_adapters(got, y, x, a, b, which, scale, at)
    assert ops.add_adapters(y, x, a, b, which, scale, inplace=True) is y and torch.equal(y, got)
