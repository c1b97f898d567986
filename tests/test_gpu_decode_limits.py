"""The operators of a decoding step at the limits of their arithmetic, against the formulas in 64 bits."""
import math

import pytest
import torch

from kernelcodegen_amd import ops
from test_gpu_decode_step import DTYPE, HALF_ULP, attention_case, close, ints, laid_out, plain_attention, plain_pages, same, values

pytestmark = pytest.mark.gpu


def near(got, expected):
    """As `close`, for values of any size: nothing is added but half the distance of the least numbers of IEEE half, 2^-25."""
    want, mag = expected
    tol = want.abs() * HALF_ULP[got.dtype] + mag * 1.25 * HALF_ULP[torch.float16] + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


def again(call):
    """The result of the second of two calls, whose memory is that of the first one's, filled with NaN."""
    call()
    first = call()
    where = first.data_ptr()
    first.fill_(math.nan)
    del first
    second = call()
    assert second.data_ptr() == where
    return second


@pytest.mark.parametrize("d", [32, 96, 128, 160, 224])
@pytest.mark.parametrize("waves,rb", [(1, 1), (1, 2), (2, 1), (2, 2)])
def test_tiles_of_fewer_wavefronts_are_joined_whole(d, waves, rb):
    lengths, counts = [900, 300], [40, 70]
    q, caches, scales, table, starts = attention_case(d + waves, lengths, counts, 4, 2, d, 16, "tokens", "bf16")
    want = plain_attention(q, *caches, *scales, table, lengths, starts, d ** -0.5, 0.0, 0, None)
    keys, first = ints(lengths), ints(starts)
    close(again(lambda: ops.cache_attention(q, *caches, *scales, table, keys, first, SHARE=1, WHOLE=0, WAVES=waves, RB=rb, GRID=50)), want)


# ---- scales far apart

def far_apart(dtype, many, low, seed=11):
    """Two requests whose pages have in turn a scale and 2^low of it; all are attended to."""
    lengths, counts = ([400, 90], [70, 20]) if many else ([400, 90, 33, 3000], None)
    q, caches, scales, table, starts = attention_case(seed, lengths, counts, 8, 2, 64, 16, "tokens", dtype, spread=0)
    held = [table[b, :-(-n // 16)].long() for b, n in enumerate(lengths)]
    return q, caches, scales, table, lengths, starts, held


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("low", [-11, -20, -24, -30, -60])
@pytest.mark.parametrize("first", [0, 1])
def test_pages_of_small_values_keep_their_weight(dtype, many, low, first):
    q, caches, scales, table, lengths, starts, held = far_apart(dtype, many, low)
    for pages in held:
        scales[1][pages[first::2]] *= 2.0 ** low
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), None if starts is None else ints(starts))
    near(got, plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, 0.0, 0, None))


@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("first", [0, 1])
def test_scales_as_far_apart_as_they_may_be(many, first):
    """A factor of 2^100, the least 2^-78."""
    q, caches, scales, table, lengths, starts, held = far_apart("bf16", many, 0, 20)
    for pages in held:
        scales[1][pages] *= 2.0 ** 30
        scales[1][pages[first::2]] *= 2.0 ** -100
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), None if starts is None else ints(starts))
    near(got, plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, 0.0, 0, None))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("count", [1, 40])
@pytest.mark.parametrize("sink", [-11, 0])
def test_many_keys_of_little_weight_beside_one_of_much(dtype, count, sink):
    """One key has 2^15 to 2^17 times the weight of each of the others, whose page's scale is 2^-11 of its own or 2^11 times that."""
    n, d = 40000, 32
    caches = [laid_out(2500, 16, 1, d, "tokens") for _ in range(2)]
    k, v = (c.view(torch.uint8) for c in caches)
    k[0, 0, 0, 0] = 0x52                      # 10
    g = torch.Generator(device="cuda").manual_seed(3)
    v.copy_(((torch.rand((2500, 16, 1, d), generator=g, device="cuda") + 0.5) * 128).to(torch.float8_e4m3fn).view(torch.uint8))
    scales = [torch.ones((2500, 1), device="cuda") for _ in range(2)]
    scales[1][1:] = 2.0 ** -11
    if sink:
        scales[1] = 2.0 ** -11 / scales[1]
    q = torch.zeros((count, 1, d), device="cuda", dtype=DTYPE[dtype])
    q[:, 0, 0] = torch.linspace(1.04, 1.18, count, device="cuda") if count > 1 else 1.11
    table = torch.arange(2500, device="cuda", dtype=torch.int32)[None]
    starts = None if count == 1 else [0, count]
    got = ops.cache_attention(q, *caches, *scales, table, ints([n]), None if starts is None else ints(starts), scale=1.0)
    near(got, plain_attention(q, *caches, *scales, table, [n], starts, 1.0, 0.0, 0, None))


# ---- pages of zeros

@pytest.mark.parametrize("dtype,size", [("bf16", 0), ("bf16", -14), ("bf16", -30), ("bf16", -50), ("f16", 0), ("f16", -12)])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("zeros", [[0], [0, 1, 2, 3], [1, 5], [2, 3, 4, 5, 6, 7, 8]])
def test_pages_of_zeros_leave_small_values_their_bits(dtype, size, many, zeros):
    """Pages of zeros stand first, or behind a page of large values that nobody attends to; V is of some size 2^size."""
    q, caches, scales, table, lengths, starts, held = far_apart(dtype, many, 0, 12)
    scales[1] *= 2.0 ** size
    for pages in held:
        scales[1][pages[[z for z in zeros if z < len(pages)]]] = 0.0
    if 0 not in zeros:
        # the request's first page: large values, and keys that the first head's queries point away from
        for b, pages in enumerate(held):
            scales[1][pages[0]] *= 2.0 ** 20
            caches[0].view(torch.uint8)[pages[0]] = 0x78 + 0x80
            scales[0][pages[0]] = 4.0
        q.abs_()
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), None if starts is None else ints(starts))
    near(got, plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, 0.0, 0, None))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("count", [1, 40])
def test_a_key_of_a_page_of_zeros_may_have_most_of_the_weight(dtype, count):
    n, d = 40000, 32
    caches = [laid_out(2500, 16, 1, d, "tokens") for _ in range(2)]
    k, v = (c.view(torch.uint8) for c in caches)
    k[0, 0, 0, 0] = 0x54                      # 12: 2^17 times the others' weight
    g = torch.Generator(device="cuda").manual_seed(4)
    v.copy_(((torch.rand((2500, 16, 1, d), generator=g, device="cuda") + 0.5) * 128).to(torch.float8_e4m3fn).view(torch.uint8))
    scales = [torch.ones((2500, 1), device="cuda") for _ in range(2)]
    scales[1].fill_(2.0 ** -8)
    scales[1][0] = 0.0
    q = torch.zeros((count, 1, d), device="cuda", dtype=DTYPE[dtype])
    q[:, 0, 0] = 1.0
    table = torch.arange(2500, device="cuda", dtype=torch.int32)[None]
    starts = None if count == 1 else [0, count]
    got = ops.cache_attention(q, *caches, *scales, table, ints([n]), None if starts is None else ints(starts), scale=1.0)
    near(got, plain_attention(q, *caches, *scales, table, [n], starts, 1.0, 0.0, 0, None))


@pytest.mark.parametrize("many", [False, True])
def test_only_pages_of_zeros(many):
    q, caches, scales, table, lengths, starts, held = far_apart("bf16", many, 0, 13)
    scales[1].zero_()
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), None if starts is None else ints(starts))
    assert not bool(got.any())


# ---- rows that see no key

def test_rows_behind_the_last_request_may_be_many():
    """More rows than 32 bits could count the keys of, if these rows had any."""
    tokens = 6_200_000
    q = torch.ones((tokens, 1, 32), device="cuda", dtype=torch.bfloat16)
    caches, scales = [laid_out(4, 16, 1, 32, "tokens") for _ in range(2)], [torch.ones((4, 1), device="cuda") for _ in range(2)]
    for c in caches:
        c.view(torch.uint8).fill_(0x38)
    table, keys, starts = ints([[0, 1, 2, 3]]), ints([64]), ints([0, 3])
    got = again(lambda: ops.cache_attention(q, *caches, *scales, table, keys, starts))
    assert bool((got[:3] == 1).all()) and not bool(got[3:].any())


@pytest.mark.parametrize("lengths,counts,pad,window", [([100, 40], [30, 1], 3000, 0), ([64], [2], 500, 0), ([10, 700], [900, 40], 20, 0), ([10, 700], [900, 40], 300, 50),
                                                       ([5, 0, 300], [200, 7, 3], 100, 1000)])
@pytest.mark.parametrize("kv_heads", [1, 4])
def test_rows_without_keys_beside_others(lengths, counts, pad, window, kv_heads):
    q, caches, scales, table, starts = attention_case(15, lengths, counts, 4, kv_heads, 64, 16, "tokens", "bf16")
    q = torch.cat([q, torch.ones_like(q[:1]).expand(pad, -1, -1)])
    want = plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, 0.0, window, None)
    keys, first = ints(lengths), ints(starts)
    for form in ({}, dict(SHARE=0, WHOLE=0, RB=1, WAVES=4, GRID=7), dict(SHARE=0, WHOLE=1, RB=1, WAVES=2), dict(SHARE=1, WHOLE=0, RB=2, WAVES=4, GRID=64)):
        got = again(lambda: ops.cache_attention(q, *caches, *scales, table, keys, first, window=window or None, **form))
        close(got, want)
        assert not bool(got[starts[-1]:].any())


# ---- infinities and NaN among zeros

@pytest.mark.parametrize("dtype", sorted(DTYPE))
def test_infinities_among_zeros_count_as_zeros(dtype):
    caches, scales = [laid_out(4, 16, 2, 64, "tokens") for _ in range(2)], [torch.full((4, 2), 7.0, device="cuda") for _ in range(2)]
    x = torch.zeros((20, 2, 64), device="cuda", dtype=DTYPE[dtype])
    x[3, 0, 5], x[18, 0, 6], x[4, 1, 7], x[19, 1, 0] = math.inf, -math.inf, math.nan, math.inf
    at = torch.arange(20, device="cuda") + 16
    ops.cache_write(x, x, *caches, *scales, at)
    # all finite magnitudes are zeros, so the scales are; a NaN stays one
    want = torch.zeros((64, 2, 64), device="cuda", dtype=torch.float64)
    want[16:36][x.isnan()] = math.nan
    assert scales[0][:, 0].tolist() == scales[1][:, 1].tolist() == [7, 0, 0, 7] and same(values(caches[0]).view(64, 2, 64), want)
    back = ops.cache_read(caches[0], scales[0], at, torch.float32)
    assert int(back.isnan().sum()) == 1 and bool(back[4, 1, 7].isnan()) and not bool(back.nan_to_num().any())
    q = torch.ones((1, 2, 64), device="cuda", dtype=torch.float16)
    got = ops.cache_attention(q, *caches, *scales, ints([[1, 2]]), ints([20]))
    assert not bool(got[0, 0].any()) and bool(got[0, 1].isnan().all())


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("many", [False, True])
def test_nan_of_a_page_of_zeros_stays(dtype, many):
    """What such a page holds times its scale is zero, or NaN where that is NaN, of K and of V."""
    q, caches, scales, table, lengths, starts, held = far_apart(dtype, many, 0, 14)
    scales[1][held[0][3]] = 0.0
    v = caches[1].view(torch.uint8)
    v[held[0][3]] &= 0x3F
    v[held[0][3], 5, 1, 9] = 0x7F
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), None if starts is None else ints(starts))
    rows = got[:70] if many else got[:1]
    assert bool(rows[:, 4:, 9].isnan().all()) and int(got.isnan().sum()) == rows.shape[0] * 4


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 40])
@pytest.mark.parametrize("lengths,counts", [([10], [30]), ([100, 7], [3, 90]), ([300, 64], [400, 70])])
def test_a_window_of_all_keys_before_rows_without_keys(window, lengths, counts):
    q, caches, scales, table, starts = attention_case(18, lengths, counts, 4, 2, 64, 16, "tokens", "bf16")
    want = plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, 0.0, 0, None)
    for form in ({}, dict(SHARE=1, WHOLE=0, RB=1, WAVES=4), dict(SHARE=0, WHOLE=0, RB=1, WAVES=4), dict(SHARE=0, WHOLE=1, RB=1, WAVES=2)):
        close(ops.cache_attention(q, *caches, *scales, table, ints(lengths), ints(starts), window=window, **form), want)


# ---- page_slots

def test_page_slots_of_no_requests():
    none, table, free = ints([]), torch.zeros((0, 3), device="cuda", dtype=torch.int32), ints([7, 8])
    for tokens in (0, 5, 3000):
        for r in ops.page_slots(none, none, table, free, 16, tokens):
            r.fill_(-9)
        slots, positions, starts, lengths, used = ops.page_slots(none, none, table, free, 16, tokens)
        assert starts.tolist() == [0] and used.tolist() == [0] and lengths.tolist() == [] and slots.tolist() == positions.tolist() == [-1] * tokens


@pytest.mark.parametrize("page", [2 ** 30, 2 ** 30 + 5, 2 ** 31 - 1])
def test_page_slots_of_very_large_pages(page):
    lengths, added, free = [0, 3, 2 ** 30, 2 ** 30 + 4], [2, 1, 3, 2], [9, 4, 5, 8]
    table = [[-5, -5, -5], [6, -5, -5], [2, -5, -5], [3, 1, -5]]
    want = plain_pages(lengths, added, table, free, page, 9)
    at = ints(table)
    got = ops.page_slots(ints(lengths), ints(added), at, ints(free), page, 9)
    for g, w in zip(got, want):
        assert g.tolist() == w
    assert at.tolist() == want[5]


def test_page_slots_of_the_largest_lengths():
    lengths, added, page = [2 ** 31 - 9, 5], [8, 2], 2 ** 26
    table = [list(range(32)), [40] + [-1] * 31]
    want = plain_pages(lengths, added, table, [50], page, 12)
    got = ops.page_slots(ints(lengths), ints(added), ints(table), ints([50]), page, 12)
    for g, w in zip(got, want):
        assert g.tolist() == w


# ---- scores

@pytest.mark.parametrize("cap", [1e3, 1e5, 1e9, 1e38, 1e300])
@pytest.mark.parametrize("count", [1, 40])
def test_a_large_cap_leaves_scores_as_they_are(cap, count):
    """A score's error: e4m3 sums and fp32 products 2^-17 of the largest sum |q k|, tanh 2^-22 of the score."""
    lengths = [300]
    q, caches, scales, table, starts = attention_case(16, lengths, None if count == 1 else [count], 4, 2, 64, 16, "tokens", "f16")
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), None if starts is None else ints(starts), cap=cap)
    near(got, plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, cap, 0, None))


# ---- bits of the probabilities

def test_rows_of_half_precision_have_the_same_bits_in_every_form():
    """The probabilities' error is that of their sum's and scores' fp32 arithmetic, not 2^-11: by the root of the mean square over all results, half an ulp
    of the results (2^-12 at most, 0.58 of it on average) and no more than a tenth beside it."""
    lengths, counts = [2000], [200]
    q, caches, scales, table, starts = attention_case(17, lengths, counts, 4, 1, 128, 16, "tokens", "f16", spread=0)
    want, _ = plain_attention(q, *caches, *scales, table, lengths, starts, 128 ** -0.5, 0.0, 0, None)
    rounded = (want.half().double() - want).norm()
    for form in ({}, dict(SHARE=0, WHOLE=0, RB=1, WAVES=4), dict(SHARE=1, WHOLE=0, RB=1, WAVES=4), dict(SHARE=1, WHOLE=0, RB=2, WAVES=4)):
        got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), ints(starts), **form)
        assert float((got.double() - want).norm() / rounded) < 1.1, form


# ---- dispatch modes

def test_modes_that_look_at_allocations_see_the_results():
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    a = torch.ones((64, 64), device="cuda", dtype=torch.bfloat16)
    args = (ints([5]), ints([1]), ints([[3, 4]]), ints([9]))
    for call in (lambda: ops.matmul(a, a), lambda: ops.page_slots(*args, 16, 1)):
        call()
        with Seen() as seen:
            call()
        assert any("empty" in name for name in seen.names)


# ---- a step of prompts and single tokens

@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_chunks_beside_single_tokens_and_padding(dtype):
    lengths = [1 + 37 * i % 500 for i in range(60)] + [700, 300]
    counts = [1] * 60 + [200, 130]
    q, caches, scales, table, starts = attention_case(19, lengths, counts, 8, 2, 64, 16, "tokens", dtype)
    q = torch.cat([q, torch.ones_like(q[:100])])
    got = ops.cache_attention(q, *caches, *scales, table, ints(lengths), ints(starts))
    close(got, plain_attention(q, *caches, *scales, table, lengths, starts, 0.125, 0.0, 0, None))
