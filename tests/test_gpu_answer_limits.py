"""Rotation into the cache, adapters and log probabilities at the limits of their arithmetic and of their forms, against the formulas in 64 bits."""
import math

import pytest
import torch

from kernelcodegen_amd import ops
from test_gpu_answer_operators import adapters_case, angles, append_case, check_adapters, check_logprobs, turned
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
    for n, digit in enumerate(values):
        digit[n::3, n::2] = 0.0           # (nothing left of one behind the others)
    x = torch.stack(values + [torch.zeros_like(values[0])] * (4 - len(digits)), -1).view(tokens, 4 * rank).to(DTYPE[dtype])
    a = torch.eye(rank, device="cuda").repeat_interleave(4, 1)[None].to(DTYPE[dtype])
    j = torch.arange(n, device="cuda") % rank
    b = torch.nn.functional.one_hot(j, rank)[None].to(DTYPE[dtype])
    y = -values[0][:, j].to(DTYPE[out])
    which, scale = ints([0] * tokens), torch.ones(1, device="cuda")
    want = (y.double() + sum(values)[:, j]).to(DTYPE[out])
    assert torch.equal(ops.add_adapters(y, x, a, b, which), want)
    assert torch.equal(ops.add_adapters(y * 0.25, x, a, b, which, scale * 0.25), want * 0.25)


# ---- add_adapters: special values ----

@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("n,rank", [(200, 16), (101, 24), (333, 64), (70, 256)])
def test_adapters_of_infinite_numbers(dtype, out, n, rank):
    """An infinity in b, or in a, makes infinities of what it meets, as in the formula, not NaN; other columns, tokens and adapters have none of it."""
    y, x, a, b, which, scale = adapters_case(n, 40, n, 64, rank, 3, dtype, out)
    which[:] = torch.arange(40, device="cuda") % 4 - 1
    x[4:10] = torch.nn.functional.one_hot(torch.arange(6, device="cuda"), 64)          # x a that 16 bits hold
    scale[1] = -1.5
    good = ops.add_adapters(y, x, a, b, which, scale)
    b[0, 3, 5], b[0, 17, 1], b[0, n - 1, rank - 1], b[0, 9, 0], b[0, 9, 7], b[1, 3, 2], b[1, 5, 4], b[2, 6, 1] = math.inf, -math.inf, math.inf, math.inf, math.inf, -math.inf, math.nan, -math.inf
    a[2, 1, 7] = b[2, 8, 3] = math.inf          # (an infinity of x a beside one of b that meets another number)
    got = ops.add_adapters(y, x, a, b, which, scale)
    want = y.double()
    for r in range(3):
        mine = which == r
        h = x[mine].double() @ a[r].double().t()
        want[mine] += float(scale[r]) * (h[:, None, :] * b[r].double()[None]).sum(-1)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[got.isinf()].double(), want[want.isinf()]) and torch.equal(got.isinf(), want.isinf())
    fine = want.isfinite()
    assert torch.equal(got[fine], good[fine]) and bool(want[which >= 0].isinf().any())


@pytest.mark.parametrize("dtype", sorted(DTYPE))
@pytest.mark.parametrize("tokens,n", [(3, 100), (90, 101), (40, 3), (1100, 200)])
def test_adapters_rows_without_one_keep_their_bits(dtype, tokens, n):
    y, x, a, b, which, scale = adapters_case(tokens, tokens, n, 64, 16, 3, "f16" if dtype == "f16" else "bf16", dtype)
    whole = torch.int32 if dtype == "f32" else torch.int16
    y.view(whole).random_(torch.iinfo(whole).min, torch.iinfo(whole).max, generator=generator(2))          # NaN of any kind, the least numbers
    y[::2, ::3] = -0.0
    which[tokens // 2:] = -1
    for inplace in (False, True):
        got = ops.add_adapters(y.clone(), x, a, b, which, scale, inplace=inplace)
        assert torch.equal(got.view(whole)[which < 0], y.view(whole)[which < 0])


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


# ---- cache_append ----

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,d,rotated", [(1, 12, 64, 32), (140, 32, 128, 128), (20, 3, 96, 96)])
def test_queries_in_fp32_are_rounded_once(interleaved, tokens, heads, d, rotated):
    """Products of fp32 numbers are exact in 64 bits, so the formula's sum there, rounded to fp32, is one number."""
    slots = [16 + i for i in range(tokens)]
    (q, k, v), caches, scales = append_case(tokens + d, slots, heads, 2, d, 16, "tokens", "f32", 12)
    positions = ints([(37 * i) % 500 for i in range(tokens)])
    table = angles(500, rotated)
    got = ops.cache_append(q, k, v, *caches, *scales, ints(slots, torch.int64), positions, table, interleaved=interleaved)
    assert torch.equal(got, turned(q, positions, table, interleaved).float())


def test_append_writes_the_same_in_a_graph_and_on_another_stream():
    """The cache and its scales, put back before each call, with other keys, values and positions in the same places."""
    slots = list(range(16, 60))
    (q, k, v), caches, scales = append_case(5, slots, 4, 2, 64, 16, "tokens", "bf16", 5)
    at, where, table = ints(slots, torch.int64), ints([i + 3 for i in range(44)]), angles(100, 64)
    held = [c.view(torch.uint8) for c in caches] + scales
    old = [h.clone() for h in held]

    def restore():
        for h, o in zip(held, old):
            h.copy_(o)

    def append():
        return ops.cache_append(q, k, v, *caches, *scales, at, where, table)

    def what(call):
        restore()
        return [t.clone() for t in (call(), *held)]
    first, side = what(append), torch.cuda.Stream()
    assert not any(torch.equal(h, o) for h, o in zip(held, old))
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = what(append)
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = append()
    for i in range(4):
        q.copy_(torch.randn(q.shape, generator=generator(i), device="cuda"))
        k.copy_(torch.randn(k.shape, generator=generator(i + 9), device="cuda") * 4.0 ** i)
        v.copy_(torch.randn(v.shape, generator=generator(i + 19), device="cuda") * 0.25 ** i)
        where.add_(7)
        want = what(append)
        recorded.zero_()
        got = what(lambda: graph.replay() or recorded)
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want)) and not torch.equal(got[0], first[0])


# ---- token_logprobs: more rows than two for each unit ----

@pytest.mark.parametrize("dtype,rows,v,top", [("bf16", 1024, 5003, 32), ("f32", 1500, 801, 5), ("bf16", 1030, 32000, 0), ("f16", 1100, 20011, 20)])
def test_log_probabilities_of_more_than_a_thousand_rows(dtype, rows, v, top):
    """The workgroups that the rule takes from 1024 rows on; rows with few numbers left, none, an infinity or a NaN among the others."""
    g = generator(rows)
    logits = (torch.randn((rows, v), generator=g, device="cuda") * 3).to(DTYPE[dtype])
    tokens = torch.randint(-1, v + 1, (rows,), generator=g, device="cuda")
    logits[3::50, 40:] = -math.inf
    logits[7::90] = -math.inf
    logits[8::91, v // 2], logits[9::92, v - 1], logits[10::93, 5:] = math.inf, math.nan, logits[10, 0]
    check_logprobs(ops.token_logprobs(logits, tokens, top), logits, tokens, top)
    x = logits[:, 3:v - 2]
    check_logprobs(ops.token_logprobs(x, tokens - 4, min(top, 7)), x, tokens - 4, min(top, 7))
