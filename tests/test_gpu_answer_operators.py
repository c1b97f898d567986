"""Rotation on the way into the cache, adapters beside a projection, and log probabilities of tokens on the device, against plain
implementations in 64 bits."""
import math

import pytest
import torch

from kernelcodegen_amd import ops
from kernelcodegen_amd._lib import KcgError
from test_gpu_decode_step import DTYPE, HALF_ULP, generator, ints, laid_out, plain_write, put, same, values

pytestmark = pytest.mark.gpu


# ---- cache_append ----

def angles(positions, rotated, base=10000.0):
    """fp32 [positions, rotated]: cosines, then sines, of pair i turned by base^(-2 i / rotated) a position."""
    rate = base ** (-torch.arange(rotated // 2, dtype=torch.float64) * 2 / rotated)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.cat((a.cos(), a.sin()), 1).float().cuda()


def turned(x, positions, table, interleaved):
    """Rows by the formula, in fp64: x cos - y sin, y cos + x sin; rows without a position unturned, NaN behind the table."""
    r = table.shape[1]
    i = torch.arange(r // 2, device="cuda")
    one, two = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    p = positions.long()
    row = table.double()[p.clamp(0, table.shape[0] - 1)]
    row = torch.where((p >= table.shape[0])[:, None], math.nan, row)
    cos, sin = row[:, None, :r // 2], row[:, None, r // 2:]
    x = x.double()
    out = x.clone()
    out[..., one], out[..., two] = x[..., one] * cos - x[..., two] * sin, x[..., two] * cos + x[..., one] * sin
    return torch.where((p < 0)[:, None, None], x, out)


def append_case(seed, slots, heads, kv_heads, d, page, order, dtype, pages):
    g = generator(seed)
    caches, scales = [], []
    for _ in range(2):
        c = laid_out(pages, page, kv_heads, d, order)
        x = torch.randn((pages, page, kv_heads, d), generator=g, device="cuda", dtype=torch.float64)
        scales.append(put(c, x * torch.exp2(torch.randint(-6, 6, (pages, 1, kv_heads, 1), generator=g, device="cuda"))))
        caches.append(c)
    rows = torch.randn((len(slots), heads + 2 * kv_heads, d), generator=g, device="cuda") * torch.exp2(torch.randint(-9, 9, (len(slots), 1, 1), generator=g, device="cuda").float())
    return rows.to(DTYPE[dtype]).split((heads, kv_heads, kv_heads), 1), caches, scales


def some_slots(seed, pages, page):
    """Single tokens in the middle, at the start and at the end of a page; runs over pages; tokens that are left out."""
    p = torch.randperm(pages, generator=generator(seed), device="cuda").tolist()
    slots = [p[0] * page + 5, -1, p[1] * page, p[2] * page + page - 1] + [p[3] * page + i for i in range(7, page)] + [p[4] * page + i for i in range(page)]
    return slots + [p[5] * page + i for i in range(3)] + [pages * page, -100] + [p[6] * page + i for i in range(1, min(page, 12))]


def check_append(q, k, v, caches, scales, slots, positions, table, interleaved):
    at, where, page = ints(slots, torch.int64), ints(positions), caches[0].shape[1]
    want_q, want_k = turned(q, where, table, interleaved), turned(k, where, table, interleaved)
    want = [plain_write(x, c, s, at, page) for x, c, s in ((want_k, caches[0], scales[0]), (v, caches[1], scales[1]))]
    valid = (at >= 0) & (at < caches[0].shape[0] * page)
    for (w, _), x in zip(want, (want_k, v)):
        # (a NaN stays one, also in a page whose scale is 0)
        row, place = at[valid] // page, at[valid] % page
        w[row, place] = torch.where(x[valid].isnan(), math.nan, w[row, place])
    got = ops.cache_append(q, k, v, *caches, *scales, at, where, table, interleaved=interleaved)
    assert got.dtype == q.dtype and got.shape == q.shape and got.is_contiguous()
    # Queries: y sin is rounded to fp32, half a step of at most 2^-24 |y sin|, the sum again, 2^-24 of it, and then to the type, half a step of its
    # own; |y sin| is at most the largest number of the row times a cosine or sine.  (Half precision's least step is 2^-24.)
    most = q.double().abs().amax(-1, keepdim=True).nan_to_num(0.0, 0.0, 0.0) * max(1.0, float(table.abs().max()))
    off = (got.double() - want_q).abs()
    fine = off <= 2.0 ** -24 * (most + want_q.abs()) + HALF_ULP[q.dtype] * (want_q.abs() + 2.0 ** -23 * most) + (2.0 ** -25 if q.dtype == torch.float16 else 0.0)
    assert bool((fine | (got.double() == want_q) | (got.isnan() & want_q.isnan())).all())
    unturned = (where < 0)[:, None, None] | (torch.arange(q.shape[2], device="cuda") >= table.shape[1])
    assert same(torch.where(unturned, got, 0.0), torch.where(unturned, q, 0.0))
    for c, s, (w, ws) in zip(caches, scales, want):
        assert torch.equal(s.double(), ws) and same(values(c), w)


@pytest.mark.parametrize("dtype", sorted(DTYPE))
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads,d,rotated,page,order", [
    (32, 8, 128, 128, 16, "tokens"), (3, 3, 64, 32, 32, "heads"), (2, 1, 96, 96, 64, "apart"), (4, 2, 256, 64, 128, "tokens"), (10, 5, 32, 16, 16, "heads"),
    (6, 2, 160, 80, 256, "tokens"), (7, 1, 224, 224, 32, "tokens")])
def test_cache_append(dtype, interleaved, heads, kv_heads, d, rotated, page, order):
    pages = 40
    slots = some_slots(heads * d, pages, page)
    (q, k, v), caches, scales = append_case(heads + d, slots, heads, kv_heads, d, page, order, dtype, pages)
    positions = [(37 * i) % 500 for i in range(len(slots))]
    positions[1], positions[2] = -1, 499
    check_append(q, k, v, caches, scales, slots, positions, angles(500, rotated), interleaved)
    if order == "apart":
        around = torch.empty(0, dtype=torch.uint8, device="cuda").set_(caches[0].untyped_storage()).view(pages, page, kv_heads + 1, 2 * d)
        assert not bool(around[:, :, kv_heads:].any()) and not bool(around[..., :d].any())


@pytest.mark.parametrize("tokens", [1, 130, 700, 2100])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_cache_append_of_many_tokens(tokens, dtype):
    """One, four and sixteen tokens to a wavefront; pages of which a wavefront's registers hold a part."""
    page, pages = 64, -(-tokens // 64) + 3
    slots = [page + 9 + i for i in range(tokens)]
    (q, k, v), caches, scales = append_case(tokens, slots, 5, 2, 64, page, "tokens", dtype, pages)
    check_append(q, k, v, caches, scales, slots, [9 + i for i in range(tokens)], angles(4000, 64), False)


def test_cache_append_without_positions_and_behind_the_table():
    slots = [16 + i for i in range(20)]
    for interleaved in (False, True):
        (q, k, v), caches, scales = append_case(3, slots, 4, 2, 64, 16, "tokens", "f16", 5)
        positions = [-1] * 5 + [99, 100, 2 ** 31 - 1, -2 ** 31] + list(range(11))
        check_append(q, k, v, caches, scales, slots, positions, angles(100, 32), interleaved)


def test_cache_append_of_far_positions_and_numbers_at_borders():
    """Sums of products that fp32 would round over a border of the 8 bits, or of 448 times a power of two."""
    slots = [16 * 3 + i for i in range(640)]
    (q, k, v), caches, scales = append_case(8, slots, 2, 2, 64, 16, "tokens", "f16", 50)
    k.copy_((torch.randint(17, 32, k.shape, generator=generator(1), device="cuda") * 2.0 - 1).half())         # ties of four binary digits
    check_append(q, k, v, caches, scales, slots, [131072 - 700 + i for i in range(640)], angles(131072, 64, 5e5), False)
    one = torch.zeros((8, 64), device="cuda")
    one[:, :32] = 1.0 + torch.arange(-3, 5, device="cuda")[:, None] * 2.0 ** -23                                   # cosines next to 1
    k.fill_(7.0)
    (q, _, v), caches, scales = append_case(9, slots, 2, 2, 64, 16, "tokens", "f16", 50)
    check_append(q, k, v, caches, scales, slots, [i // 16 % 8 for i in range(640)], one, False)


def test_cache_append_of_infinities_and_zeros():
    slots = [16 + i for i in range(4)]
    (q, k, v), caches, scales = append_case(5, slots, 2, 2, 64, 16, "tokens", "bf16", 4)
    k.zero_()
    k[1, 0, 40], k[2, 1, 60], k[3, 1, 3] = math.inf, -math.inf, math.nan        # (the last 32 are not turned)
    v[2, 0, 1] = math.inf
    check_append(q, k, v, caches, scales, slots, [5, 6, 7, 8], angles(10, 32), False)


def test_cache_append_offsets_beyond_32_bits():
    """Pages behind 2^31 bytes of the cache, and rows of queries, keys and values that lie 2^29 numbers apart."""
    page, heads, d, pages = 16, 8, 256, 70000
    caches, scales = [torch.zeros((pages, page, heads, d), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)], [torch.zeros((pages, heads), device="cuda") for _ in range(2)]
    far = torch.empty((6, 1 << 29), device="cuda", dtype=torch.bfloat16)
    rows = far[:, :(4 + 2 * heads) * d].view(6, 4 + 2 * heads, d)
    rows.copy_(torch.randn(rows.shape, generator=generator(4), device="cuda"))
    q, k, v = rows.split((4, heads, heads), 1)
    slots, where, table = [page * 7 + page - 1, page * 7 + 1, page * 5, page * 5 + 1, page * 5 + 2, -1], ints([3, 900, 0, 1, 2, 5]), angles(1000, 64)
    at = ints(slots, torch.int64)
    want_q, want_k = turned(q, where, table, False), turned(k, where, table, False)
    want = [plain_write(x, c[-8:], s[-8:], at, page) for x, c, s in ((want_k, caches[0], scales[0]), (v, caches[1], scales[1]))]
    got = ops.cache_append(q, k, v, *caches, *scales, torch.where(at < 0, at, at + (pages - 8) * page), where, table)
    assert bool(((got.double() - want_q).abs() <= 2.0 ** -8 * want_q.abs() + 2.0 ** -20).all())       # (half a step, and the sums' 2^-23 of numbers below 8)
    for c, s, (w, ws) in zip(caches, scales, want):
        assert torch.equal(s[-8:].double(), ws) and same(values(c[-8:]), w) and not bool(s[:-8].any()) and not bool(c[:-8].view(torch.uint8).any())


def test_cache_append_then_attention_sees_distances_only():
    """Rotated queries and keys: scores go by the distance, so a prompt moved along the positions has the same answers."""
    d, page, tokens = 64, 16, 40
    g = generator(4)
    qkv = torch.randn((tokens, 8, d), generator=g, device="cuda").half()
    q, k, v = qkv.split((4, 2, 2), 1)
    table = angles(5000, d)
    outs = []
    for start in (0, 4000):
        caches, scales = [laid_out(4, page, 2, d, "tokens") for _ in range(2)], [torch.zeros((4, 2), device="cuda") for _ in range(2)]
        slots = torch.arange(tokens, device="cuda")
        turned_q = ops.cache_append(q, k, v, *caches, *scales, slots, torch.arange(start, start + tokens, device="cuda", dtype=torch.int32), table)
        outs.append(ops.cache_attention(turned_q, *caches, *scales, ints([[0, 1, 2]]), ints([tokens]), ints([0, tokens])))
    # each key is off by 2^-4 of its size, a score (64 products, d^-1/2) by about 2^-4 of 1 standard deviation
    assert float((outs[0] - outs[1]).abs().max()) < 0.35 and not torch.equal(outs[0], outs[1])


# ---- add_adapters ----

def adapters_case(seed, tokens, n, k, rank, adapters, dtype, out, spread=1.0):
    g = generator(seed)
    x = torch.randn((tokens, k), generator=g, device="cuda").to(DTYPE[dtype])
    y = torch.randn((tokens, n), generator=g, device="cuda").to(DTYPE[out])
    a = (torch.randn((adapters, rank, k), generator=g, device="cuda") * k ** -0.5 * spread).to(DTYPE[dtype])
    b = (torch.randn((adapters, n, rank), generator=g, device="cuda") * 0.3).to(DTYPE[dtype])
    which = torch.randint(-1, adapters, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    return y, x, a, b, which, torch.rand(adapters, generator=g, device="cuda") * 2


def check_adapters(got, y, x, a, b, which, scale, at=slice(None)):
    """`at`: the tokens to look at."""
    rank, k = a.shape[1:]
    y, x, which = y[at], x[at], which[at]
    want, mag_x, mag_h = y.double(), torch.zeros(y.shape, dtype=torch.float64, device="cuda"), torch.zeros(y.shape, dtype=torch.float64, device="cuda")
    for r in set(which.tolist()):
        if not 0 <= r < a.shape[0]:
            continue
        mine = which == r
        by = 1.0 if scale is None else abs(float(scale[r]))
        h = x[mine].double() @ a[r].double().t()
        want[mine] += (1.0 if scale is None else float(scale[r])) * (h @ b[r].double().t())
        mag_x[mine] = by * ((x[mine].double().abs() @ a[r].double().abs().t()) @ b[r].double().abs().t())
        mag_h[mine] = by * (h.abs() @ b[r].double().abs().t())
    # sums of k: 32 numbers in an instruction, then one instruction after the other; of the rank's, three times; h as a sum of 16-bit numbers: 2^-16 of it
    # with two of bfloat16, for results in that, 2^-20 with two of half precision, all of it with three; the scales' product and the sum with y in fp32
    eps = 2.0 ** -24
    kept = 2.0 ** -20 if x.dtype == torch.float16 else 0.0 if y.dtype == torch.float32 else 2.0 ** -16
    tol = mag_x * (k / 32 + 64) * eps + mag_h * ((3 * rank / 32 + 40) * eps + kept) + \
        (want.abs() + mag_h) * 4 * eps + want.abs() * HALF_ULP[y.dtype] + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    off = (got[at].double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol.clamp(min=1e-300)).max())
    none = (which < 0) | (which >= a.shape[0])
    assert torch.equal(got[at][none], y[none])


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("tokens,n,k,rank,adapters", [
    (1, 4096, 4096, 16, 8), (1, 1, 8, 8, 1), (3, 100, 520, 8, 2), (16, 513, 256, 24, 40), (17, 64, 4104, 16, 3), (64, 1000, 1000, 16, 64), (100, 333, 2048, 32, 5),
    (257, 640, 512, 64, 4), (1000, 200, 264, 128, 2), (70, 130, 96, 256, 9), (33, 71, 40, 40, 6)])
def test_add_adapters(dtype, out, tokens, n, k, rank, adapters):
    y, x, a, b, which, scale = adapters_case(tokens + n, tokens, n, k, rank, adapters, dtype, out)
    before = y.clone()
    got = ops.add_adapters(y, x, a, b, which, scale)
    assert got.dtype == y.dtype and got.is_contiguous() and torch.equal(y, before)
    check_adapters(got, y, x, a, b, which, scale)
    plain = ops.add_adapters(y, x, a, b, which)
    check_adapters(plain, y, x, a, b, which, None)
    assert ops.add_adapters(y, x, a, b, which, scale, inplace=True) is y and torch.equal(y, got)


@pytest.mark.parametrize("pattern", ["one", "runs", "all different", "none", "out of range"])
@pytest.mark.parametrize("tokens", [20, 300])
def test_add_adapters_by_who_has_which(pattern, tokens):
    adapters = 320
    y, x, a, b, which, scale = adapters_case(7, tokens, 192, 128, 16, adapters, "bf16", "bf16")
    i = torch.arange(tokens, device="cuda", dtype=torch.int32)
    which = {"one": i * 0 + 3, "runs": i // 37, "all different": adapters - 1 - i, "none": i * 0 - 1,
             "out of range": torch.where(i % 3 == 0, 2 ** 31 - 1, torch.where(i % 3 == 1, -2 ** 31, adapters)).int()}[pattern].contiguous()
    check_adapters(ops.add_adapters(y, x, a, b, which, scale), y, x, a, b, which, scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("inplace", [False, True])
def test_add_adapters_of_rows_that_lie_apart(dtype, inplace):
    """One of three projections that lie side by side; what is beside it stays."""
    y, x, a, b, which, scale = adapters_case(12, 50, 100, 256, 16, 7, dtype, dtype)
    for first in (0, 3, 104):
        all_y = torch.randn((50, 300), device="cuda").to(y.dtype)
        wide_x = torch.randn((50, 512), device="cuda").to(x.dtype)
        mine, xs, kept = all_y[:, first:first + 100], wide_x[:, 128:384], all_y.clone()
        got = ops.add_adapters(mine, xs, a, b, which, scale, inplace=inplace)
        check_adapters(got, kept[:, first:first + 100], xs, a, b, which, scale)
        if inplace:
            kept[:, first:first + 100] = got
        assert torch.equal(all_y, kept)


@pytest.mark.parametrize("dtype,out", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("ts,ut,rank", [(1, 1, 16), (2, 2, 8), (4, 4, 24), (4, 1, 64), (2, 2, 128), (4, 2, 16), (1, 4, 256), (1, 1, 40)])
@pytest.mark.parametrize("form", [dict(KS=1, S=1, NS=1), dict(KS=5, S=3, NS=2), dict(KS=8, S=16, NS=7)])
def test_add_adapters_forms(dtype, out, ts, ut, rank, form):
    """Tiles whose adapters are shared out between workgroups, or one workgroup's; parts of k, the last of which are empty."""
    y, x, a, b, which, scale = adapters_case(ts + rank, 150, 328, 1032, rank, 9, dtype, out)
    which[40:120] = 4
    check_adapters(ops.add_adapters(y, x, a, b, which, scale, TS=ts, UT=ut, **form), y, x, a, b, which, scale)
    got = ops.add_adapters(y.clone(), x, a, b, which, None, inplace=True, TS=ts, UT=ut, **form)
    check_adapters(got, y, x, a, b, which, None)


@pytest.mark.parametrize("n", [2048, 2003])
@pytest.mark.parametrize("form", [dict(S=1, NS=1), dict(S=1, NS=100), dict(S=3, NS=2), dict(UT=4, S=1, NS=3), dict(UT=2, S=2, NS=100)])
def test_add_adapters_in_place_by_passes_and_turns(n, form):
    """Tiles of many adapters, one after the other and in several passes over the columns, write what they read."""
    y, x, a, b, which, scale = adapters_case(n, 150, n, 264, 24, 11, "bf16", "bf16")
    want = ops.add_adapters(y, x, a, b, which, scale)
    assert ops.add_adapters(y, x, a, b, which, scale, inplace=True, KS=1, TS=1, **form) is y
    check_adapters(want, *adapters_case(n, 150, n, 264, 24, 11, "bf16", "bf16"))
    assert torch.equal(y, want)


def test_add_adapters_keeps_what_half_precision_would_lose():
    """x a of 2^20 and of 2^-30, which half precision holds no numbers for."""
    for spread, b_spread in ((2.0 ** 13, 2.0 ** -14), (2.0 ** -12, 1.0)):
        y, x, a, b, which, scale = adapters_case(3, 40, 128, 64, 16, 4, "f16", "f32", spread)
        b = (b * b_spread).half()
        x = (x * (64 if spread > 1 else 2.0 ** -12)).half()
        y.mul_(spread * 64 * b_spread if spread > 1 else 2.0 ** -30)
        check_adapters(ops.add_adapters(y, x, a, b, which, scale), y, x, a, b, which, scale)


def test_add_adapters_keeps_infinities_and_nan_to_their_rows():
    y, x, a, b, which, scale = adapters_case(5, 40, 64, 64, 16, 3, "bf16", "bf16")
    which[:] = torch.arange(40, device="cuda") % 4 - 1
    good = ops.add_adapters(y, x, a, b, which, scale)
    x[5, 7], x[9, 0], x[12, 3] = math.inf, math.nan, math.inf            # rows of adapters 0, 0 and none
    a[2, 3, 4] = math.nan
    got = ops.add_adapters(y, x, a, b, which, scale)
    touched = (which == 2) | torch.isin(torch.arange(40, device="cuda"), ints([5, 9]))
    assert torch.equal(got[~touched], good[~touched]) and bool(got[which == 2].isnan().all()) and not bool(got[5].isfinite().any()) and bool(got[9].isnan().all())


def test_add_adapters_offsets_beyond_32_bits():
    """A pool of more than 2^31 numbers."""
    rank, k, n, adapters = 64, 8192, 64, 4200
    a = torch.zeros((adapters, rank, k), device="cuda", dtype=torch.bfloat16)
    b = torch.zeros((adapters, n, rank), device="cuda", dtype=torch.bfloat16)
    y, x, small_a, small_b, _, _ = adapters_case(2, 3, n, k, rank, 2, "bf16", "f32")
    a[-1], a[4100], b[-1], b[4100] = small_a[0], small_a[1], small_b[0], small_b[1]
    got = ops.add_adapters(y, x, a, b, ints([adapters - 1, 4100, 5]))
    check_adapters(got, y, x, small_a, small_b, ints([0, 1, -1]), None)


def test_add_adapters_to_what_it_reads():
    """In place, x the same tensor as y."""
    _, x, a, b, which, scale = adapters_case(3, 50, 512, 512, 16, 5, "f16", "f16")
    want = ops.add_adapters(x, x, a, b, which, scale)
    y = x.clone()
    assert ops.add_adapters(y, y, a, b, which, scale, inplace=True) is y and torch.equal(y, want)


# ---- token_logprobs ----

def check_logprobs(got, logits, tokens, top, terms=600):
    """`terms`: numbers that one lane may add up in turn."""
    logprob, entropy, values_, indices = got
    x = logits.double()
    rows, v = x.shape
    assert logprob.shape == entropy.shape == (rows,) and values_.shape == indices.shape == (rows, top)
    m = x.amax(-1, keepdim=True)
    broken = (x.isnan() | (x == math.inf)).any(-1)
    empty = (x == -math.inf).all(-1)
    d = torch.where((broken | empty)[:, None], 0.0, x - m)
    e = torch.exp(d)
    s = e.sum(-1, keepdim=True)
    spread = torch.where(e > 0, d * e, 0.0).sum(-1) / s[:, 0]
    want = d - s.log()
    want_entropy = s.log()[:, 0] - spread
    # each e is off by 2^-23 and 1.5 |d| 2^-24 of it, a lane's sum by its number of terms, ln s by what s is off of its size; then two roundings
    eps = 2.0 ** -24
    rel = (terms + 1.5 * spread.abs() + 20) * eps

    def close(a, b, more=0.0):
        fine = ((a.double() - b).abs() <= rel[:, None] + more * eps + 3 * b.abs() * eps) | (a.double() == b)
        assert bool((fine | (broken | empty)[:, None]).all())
        assert bool((a[broken].isnan()).all()) and bool((a[empty] == -math.inf).all())

    inside = (tokens >= 0) & (tokens < v)
    mine = torch.where(inside[:, None], want.gather(1, tokens.clamp(0, v - 1)[:, None]), -math.inf)
    close(logprob[:, None], mine)
    h = (entropy.double() - want_entropy).abs() <= rel * (2 + spread.abs()) + 4 * want_entropy.abs() * eps
    assert bool((h | broken | empty).all()) and bool(entropy[broken].isnan().all()) and bool((entropy[empty] == 0).all())
    assert bool((entropy[~broken] >= 0).all())
    ordered = torch.where(logits.isnan(), -math.inf, logits.float())
    order = torch.sort(ordered, dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(indices, order)
    close(values_, want.gather(1, order))


@pytest.mark.parametrize("dtype", sorted(DTYPE))
@pytest.mark.parametrize("rows,v,top", [
    (1, 1, 1), (1, 7, 7), (5, 100, 0), (2, 1000, 32), (64, 4096, 5), (3, 32000, 20), (300, 5003, 3), (7, 50021, 10), (1, 128000, 32), (260, 131, 31), (1, 262147, 8),
    (2, 524288, 4)])
def test_token_logprobs(dtype, rows, v, top):
    g = generator(rows + v)
    logits = (torch.randn((rows, v), generator=g, device="cuda") * 4).to(DTYPE[dtype])
    tokens = torch.randint(0, v, (rows,), generator=g, device="cuda")
    tokens[0] = logits[0].float().argmax()
    if rows > 2:
        tokens[1], tokens[2] = -1, v
    check_logprobs(ops.token_logprobs(logits, tokens, top), logits, tokens, top, 600 + v // 256)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("parts", [1, 2, 5, 16])
@pytest.mark.parametrize("threads", [64, 256, 1024])
def test_token_logprobs_forms_agree(dtype, parts, threads):
    g = generator(parts)
    logits = (torch.randn((6, 20011), generator=g, device="cuda") * 2).to(DTYPE[dtype])
    tokens = torch.randint(0, 20011, (6,), generator=g, device="cuda")
    check_logprobs(ops.token_logprobs(logits, tokens, 9, PARTS=parts, THREADS=threads), logits, tokens, 9, 1000)
    check_logprobs(ops.token_logprobs(logits[:, 3:20000], tokens % 19000, 0, PARTS=parts, THREADS=threads), logits[:, 3:20000], tokens % 19000, 0, 1000)


@pytest.mark.parametrize("dtype", sorted(DTYPE))
@pytest.mark.parametrize("rows", [3, 400])
def test_token_logprobs_of_ties_and_orders(dtype, rows):
    """All equal; rising; falling; a few values; the largest ones all in one vector, or one in each segment."""
    v, t = 9001, DTYPE[dtype]
    i = torch.arange(v, device="cuda")
    kinds = [torch.full((v,), 2.5), i / 64.0, -i / 64.0, (i * 7919 % 5).float(), torch.where(i // 8 == 500, 9.0 + i % 8, i % 3 * 1.0), torch.where(i % 128 == 77, 5.0, 0.0),
             torch.where(i % 2 == 0, -0.0, 0.0), torch.full((v,), torch.finfo(t).min), torch.where(i < 4, 1.0, -math.inf)]
    for at, kind in enumerate(kinds):
        logits = kind.to("cuda").to(t).expand(rows, v).contiguous()
        tokens = (torch.arange(rows, device="cuda") * 31) % v
        for top in (1, 20):
            check_logprobs(ops.token_logprobs(logits, tokens, top), logits, tokens, top, 600)


@pytest.mark.parametrize("dtype", sorted(DTYPE))
@pytest.mark.parametrize("parts", [1, 3])
def test_token_logprobs_of_masks_infinities_and_nan(dtype, parts):
    v, t = 7000, DTYPE[dtype]
    logits = torch.randn((12, v), generator=generator(2), device="cuda").to(t)
    logits[0] = -math.inf
    logits[1, 100:] = -math.inf
    logits[2, :6900] = -math.inf
    logits[3, 17] = math.inf
    logits[4, 6999] = math.nan
    logits[5] = math.nan
    logits[6, :] = torch.finfo(t).min
    logits[6, 5000] = 0.0
    logits[7, 3] = torch.finfo(t).max
    logits[8] = -math.inf
    logits[8, 4321] = torch.finfo(t).min
    logits[9, 40:] = torch.finfo(t).min
    logits[10] = -math.inf
    logits[10, 1], logits[10, 2] = math.inf, math.nan
    tokens = ints([0, 5000, 6950, 17, 5, 5, 5000, 3, 4321, 6000, 1, -5], torch.int64)
    check_logprobs(ops.token_logprobs(logits, tokens, 12, PARTS=parts), logits, tokens, 12)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_token_logprobs_of_large_numbers(dtype):
    """Rows around numbers of any size and sign, which are apart by single steps of the type, a few, or as usual."""
    g = generator(12)
    around = [3.0, 1e3, 1e6, 2.0 ** 23, 2.0 ** 29, 2.0 ** 30 * (1 - 2.0 ** -24), 2.0 ** 30, 2.0 ** 31, 1e12, 1e38, 3e38]
    at = torch.tensor(around + [-x for x in around], device="cuda").to(DTYPE[dtype])
    step = torch.frexp(at.float()).exponent - (24 if dtype == "f32" else 8)
    n = torch.randint(-9, 10, (len(at), 5003), generator=g, device="cuda")
    logits = torch.cat([(at.double()[:, None] + n * m * torch.exp2(step.double())[:, None]) for m in (1, 7, 300)] + [at.double()[:, None] + n.double()]).to(DTYPE[dtype])
    tokens = torch.randint(0, 5003, (len(logits),), generator=g, device="cuda")
    for parts in (1, 3):
        check_logprobs(ops.token_logprobs(logits, tokens, 4, PARTS=parts), logits, tokens, 4)
    logits[:, ::3] = -math.inf
    check_logprobs(ops.token_logprobs(logits, tokens, 4), logits, tokens, 4)


def test_token_logprobs_of_rows_that_lie_apart_and_are_alike():
    wide = torch.randn((20, 6000), generator=generator(1), device="cuda").half()
    tokens = torch.arange(10, device="cuda") * 17
    for x in (wide[::2, 5:5000], wide[:10, 8:4008], wide[:1, :3000].expand(10, 3000), wide[3:13, 1:2]):
        t = tokens % x.shape[1]
        check_logprobs(ops.token_logprobs(x, t, 1), x, t, 1)
    far = torch.zeros((3, 1 << 30), device="cuda", dtype=torch.bfloat16)        # rows more than 2^31 bytes apart
    far[:, 11:3011] = torch.randn((3, 3000), generator=generator(6), device="cuda").bfloat16()
    check_logprobs(ops.token_logprobs(far[:, 11:3011], tokens[:3], 5), far[:, 11:3011], tokens[:3], 5)


# ---- what is refused, other streams, nothing to do ----

@pytest.mark.parametrize("parts", [1, 3])
def test_token_logprobs_offsets_beyond_32_bits(parts):
    far = torch.empty((4, (1 << 30) + 5), device="cuda", dtype=torch.bfloat16)
    logits = far[:, :20011]
    logits.copy_(torch.randn(logits.shape, generator=generator(9), device="cuda") * 3)
    tokens = ints([0, 20010, 7, 20011], torch.int64)
    check_logprobs(ops.token_logprobs(logits, tokens, 6, PARTS=parts), logits, tokens, 6)


def refused(call, good, bads):
    call(**good)
    for bad in bads:
        with pytest.raises((ValueError, TypeError, KcgError)):
            call(**{**good, **bad})


def test_refusals():
    page, d = 16, 64
    kc, vc = (laid_out(4, page, 2, d, "tokens") for _ in range(2))
    ks, vs = torch.ones((4, 2), device="cuda"), torch.ones((4, 2), device="cuda")
    q = torch.ones((1, 4, d), device="cuda", dtype=torch.float16)
    k, slots, positions, table = q[:, :2], ints([3], torch.int64), ints([3]), angles(5, 32)
    shifted = torch.ones(1 + 4 * d, device="cuda", dtype=torch.float16)[1:].view(1, 4, d)
    refused(ops.cache_append, dict(q=q, k=k, v=k, k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, slots=slots, positions=positions, rotation=table),
            [dict(q=q.float()), dict(q=q.cpu()), dict(q=q[..., :32]), dict(q=q[0]), dict(q=shifted), dict(q=q[:, :0]), dict(q=q.expand(2, 4, d)), dict(k=q, v=q), dict(v=k.float()),
             dict(k=k.double(), v=k.double()), dict(k_cache=kc[:2]), dict(k_cache=kc.view(torch.uint8)), dict(k_scale=ks.cpu()), dict(v_scale=vs[:3]), dict(slots=slots.int()),
             dict(slots=ints([1, 2], torch.int64)), dict(positions=positions.long()), dict(positions=ints([1, 2])), dict(positions=positions.cpu()), dict(positions=positions[None]),
             dict(rotation=table.double()), dict(rotation=table.half()), dict(rotation=table[:0]), dict(rotation=table[0]), dict(rotation=angles(5, 24)), dict(rotation=angles(5, 80)),
             dict(rotation=table.cpu()), dict(rotation=table[:, :16]), dict(rotation=torch.ones(161, device="cuda")[1:].view(5, 32))])
    y, x, a, b, which, scale = adapters_case(1, 3, 40, 64, 8, 2, "f16", "f16")
    refused(ops.add_adapters, dict(y=y, x=x, a=a, b=b, which=which, scale=scale),
            [dict(y=y.bfloat16()), dict(y=y.double()), dict(x=x.float()), dict(x=x.float(), a=a.float(), b=b.float(), y=y.float()), dict(a=a.bfloat16()), dict(b=b.float()), dict(y=y[:2]),
             dict(x=x[:, :56]), dict(x=x[:2]), dict(a=a[:1]), dict(b=b[:1]), dict(b=b[:, :39]), dict(a=a[:0], b=b[:0], scale=scale[:0]), dict(which=which.long()), dict(which=which[:2]),
             dict(which=which.cpu()), dict(scale=scale[:1]), dict(scale=scale.half()), dict(scale=scale.cpu()), dict(x=x.cpu()), dict(a=a.cpu()), dict(y=y.cpu()), dict(a=a[:, :4], b=b[..., :4]),
             dict(a=a[:, :4].contiguous(), b=b[..., :4].contiguous()), dict(a=a.transpose(1, 2)), dict(x=x[:, :36].contiguous(), a=a[..., :36].contiguous()), dict(x=x.t().contiguous().t()),
             dict(y=y.t().contiguous().t()), dict(x=torch.ones(200, device="cuda", dtype=torch.half)[4:196].view(3, 64)), dict(y=y[:1].expand(3, 40), inplace=True), dict(KS=65), dict(PARTS=2), dict(S=0), dict(TS=3)])
    logits, tokens = torch.ones((3, 50), device="cuda"), ints([1, 2, 3], torch.int64)
    refused(ops.token_logprobs, dict(logits=logits, tokens=tokens, top=3),
            [dict(logits=logits.double()), dict(logits=logits.cpu()), dict(logits=logits[0]), dict(logits=logits[:2]), dict(logits=logits[:, :0], top=0), dict(logits=logits.t().contiguous().t()),
             dict(logits=torch.ones((3, (1 << 19) + 1), device="cuda")), dict(tokens=tokens.int()), dict(tokens=tokens.cpu()), dict(tokens=tokens[None]), dict(top=33), dict(top=-1), dict(top=1.5),
             dict(logits=logits[:, :2], top=3), dict(PARTS=0), dict(KS=1)])


def test_nothing_to_do():
    kc, vc = (laid_out(4, 16, 2, 64, "tokens") for _ in range(2))
    ks = torch.ones((4, 2), device="cuda")
    q = torch.ones((0, 4, 64), device="cuda", dtype=torch.float16)
    assert ops.cache_append(q, q[:, :2], q[:, :2], kc, vc, ks, ks, ints([], torch.int64), ints([]), angles(3, 64)).shape == (0, 4, 64)
    y, x, a, b, which, _ = adapters_case(1, 3, 40, 64, 8, 2, "f16", "f16")
    assert ops.add_adapters(y[:0], x[:0], a, b, which[:0]).shape == (0, 40)
    out = ops.token_logprobs(torch.ones((0, 50), device="cuda"), ints([], torch.int64), 4)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 4), (0, 4)] and out[3].dtype == torch.int64


def test_other_streams_and_a_graph():
    """Several calls of each on another stream, and recorded and replayed beside eager ones."""
    slots = list(range(16, 60))
    (q, k, v), caches, scales = append_case(5, slots, 4, 2, 64, 16, "tokens", "bf16", 5)
    at, where, table = ints(slots, torch.int64), ints([i + 3 for i in range(44)]), angles(100, 64)
    y, x, a, b, which, scale = adapters_case(6, 44, 300, 256, 16, 5, "bf16", "bf16")
    logits, tokens = (torch.randn((44, 20000), generator=generator(1), device="cuda") * 3), torch.arange(44, device="cuda")

    def step():
        return (ops.cache_append(q, k, v, *caches, *scales, at, where, table), ops.add_adapters(y, x, a, b, which, scale), *ops.token_logprobs(logits, tokens, 7))
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = [step() for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(g, w) for gs in got for g, w in zip(gs, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = step()
    for i in range(4):
        # other inputs in the same places
        x.copy_(torch.randn(x.shape, generator=generator(i), device="cuda"))
        which.copy_(torch.randint(-1, 5, (44,), generator=generator(i), device="cuda"))
        q.copy_(torch.randn(q.shape, generator=generator(i), device="cuda"))
        logits.add_(torch.randn((1, 20000), generator=generator(i), device="cuda"))
        want = [w.clone() for w in step()]
        for r in recorded:
            r.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(recorded, want))


def test_results_in_inference_mode_and_of_operands_with_gradients():
    y, x, a, b, which, scale = adapters_case(1, 5, 40, 64, 8, 2, "f16", "f16")
    logits = torch.randn((5, 300), generator=generator(2), device="cuda")
    want = ops.add_adapters(y, x, a, b, which), *ops.token_logprobs(logits, which.long(), 2)
    with torch.inference_mode():
        got = ops.add_adapters(y, x, a, b, which), *ops.token_logprobs(logits, which.long(), 2)
    assert all(torch.equal(g, w) for g, w in zip(got, want))
    got = ops.add_adapters(y, x.clone().requires_grad_(), a, b, which), *ops.token_logprobs(logits.clone().requires_grad_(), which.long(), 2)
    assert all(torch.equal(g, w) and not g.requires_grad for g, w in zip(got, want))


# ---- all of them in a model ----

def test_a_layer_with_positions_and_adapters_against_the_formulas():
    from kernelcodegen_amd.decode import Decoder
    model = Decoder(3, layers=1, heads=4, kv_heads=2, d=32, wide=128, vocab=96, group=32, pages=16, width=4, seed=5, rotated=16, adapters=2, rank=8)
    added, which = [20, 1, 9], [1, -1, 0]
    tokens = torch.arange(30, device="cuda") * 3
    scores = model.step(tokens, ints(added), ints(which))
    layer, got = model.layers[0], scores.double()
    of = torch.tensor([r for r, n in zip(which, added) for _ in range(n)], device="cuda")
    positions = torch.cat([torch.arange(n, device="cuda", dtype=torch.int32) for n in added])

    def product(x, w, scale, zero):
        code = torch.stack((w & 15, w >> 4), -1).view(w.shape[0], -1, 32).double()
        return x @ ((code - zero.double()[..., None]) * scale.double()[..., None]).view(w.shape[0], -1).t()

    def adapted(x, name):
        a, b = [m.double() for m in layer["adapters"][name]]
        out = product(x, *layer[name])
        for r in range(2):
            out[of == r] += x[of == r] @ a[r].t() @ b[r].t()
        return out

    def norm(x):
        return (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()

    x, heads, first = model.embedding.double()[tokens], [], 0
    qkv = adapted(norm(x), "qkv").view(30, 8, 32)
    q, keys = turned(qkv[:, :4], positions, model.rotation, False), turned(qkv[:, 4:6], positions, model.rotation, False)
    for b, n in enumerate(added):
        at = torch.tensor([int(model.table[b, t // 16]) * 16 + t % 16 for t in range(n)], device="cuda")
        k, v = [ops.cache_read(*layer[name], at, torch.float32).double() for name in ("keys", "values")]
        # the keys in the cache are these in 8 bits: off by 2^-4 of their size at most, the smallest by 2^-10 of the scale, 448 of which hold the largest
        mine = keys[first:first + n]
        assert bool(((k - mine).abs() <= 2.0 ** -4 * mine.abs() + mine.abs().amax() * 2.0 ** -10).all())
        s = (q[first:first + n, None] * k.repeat_interleave(2, 1)[None]).sum(-1) / math.sqrt(32)
        t = torch.arange(n, device="cuda")
        s = s.masked_fill((t[None] > t[:, None])[:, :, None], -math.inf).softmax(1)
        heads.append((s[..., None] * v.repeat_interleave(2, 1)[None]).sum(1))
        first += n
    x = x + adapted(torch.cat(heads).view(30, 128), "out")
    x = x + product(torch.nn.functional.gelu(product(norm(x), *layer["up"]), approximate="tanh"), *layer["down"])
    want = product(norm(x), *model.head)[[19, 20, 29]]
    # Fourteen results follow one another, each rounded to 11 bits (2^-11 of its size at most, about a third of it in the root of the mean
    # square); none is larger than a few times what it is added to.  2^-7 is 16 whole ones.
    assert float((got - want).norm() / want.norm()) < 2.0 ** -7
    chosen, worth = model.choose(scores, 3)
    assert torch.equal(chosen, worth[3][:, 0]) and torch.equal(worth[0], worth[2][:, 0])
    check_logprobs(worth, scores, chosen, 3)


def test_a_model_with_positions_and_adapters_answers_the_same_from_a_graph():
    from kernelcodegen_amd.decode import Decoder
    prompts = [[5, 9, 200, 3] * 7, [1], [77] * 16, list(range(33))]
    made = dict(layers=2, heads=8, kv_heads=2, d=64, wide=512, vocab=256, pages=48, width=8, seed=3, rotated=64, adapters=2)
    which, runs = ints([1, 0, -1, 1]), []
    for recorded in (False, True):
        model, told = Decoder(4, **made), []
        tokens, worth = model.choose(model.step(torch.cat([torch.tensor(p, device="cuda") for p in prompts]), ints([len(p) for p in prompts]), which), 4)
        graph = None
        for i in range(16):
            if recorded and i == 1:
                graph, left = model.record(tokens, which, 4)
            if graph is None:
                chosen, worth = model.choose(model.step(tokens, which=which), 4)
                tokens.copy_(chosen)
            else:
                graph.replay()
                torch.cuda.synchronize()
                worth = [w.clone() for w in left]
            told.append((tokens.clone(), *worth))
        runs.append(told)
    assert all(torch.equal(a, b) for one, two in zip(*runs) for a, b in zip(one, two))
    # adapters and positions have an effect
    other = Decoder(4, **made)
    other.step(torch.cat([torch.tensor(p, device="cuda") for p in prompts]), ints([len(p) for p in prompts]), which)
    scores = other.step(runs[0][0][0], which=ints([0, 0, -1, 1]))
    same_ = Decoder(4, **made)
    same_.step(torch.cat([torch.tensor(p, device="cuda") for p in prompts]), ints([len(p) for p in prompts]), which)
    again = same_.step(runs[0][0][0], which=which)
    assert not torch.equal(scores[0], again[0]) and torch.equal(scores[1:], again[1:])
