"""Performance cases of the operators of a decoding step: pages, the 8-bit cache, attention over it, products with 4-bit weights.

    pages      page tables and slots of the tokens of one step, from the requests' lengths
    cache      the step's keys and values written into the cache in 8 bits with a scale for each page and head, and the pages that
               this touched read back
    attention  queries over the cache: one token per request, a few (drafts), or a chunk of a prompt; capped scores, a bias that
               grows with distance, a window
    linear     activations of a few tokens times 4-bit weights with group scales

`own` False computes them in elementary torch operations, True through `kernelcodegen_amd.ops`.
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one decode step of 64 requests: a token each, a page now and then
        dict(name="pages_decode", kind="pages", batch=64, longest=2000, most=1, page=16),
        # prompts and decodes in one step: many pages at once
        dict(name="pages_prompts", kind="pages", batch=200, longest=1500, most=700, page=32),
        # that decode step's keys and values; the page is read, enlarged and written
        dict(name="cache_decode", kind="cache", batch=64, longest=2000, most=1, page=16, heads=8, d=128, dtype="bf16", heads_first=False),
        # a few short answers of a small model in fp32, pages head by head
        dict(name="cache_small", kind="cache", batch=3, longest=77, most=5, page=32, heads=12, d=64, dtype="f32", heads_first=True),
        # prompts: whole pages at a time
        dict(name="cache_prompts", kind="cache", batch=9, longest=2048, most=2048, page=16, heads=8, d=128, dtype="f16", heads_first=False),
        # one request at the start of its answer: latency
        dict(name="attention_short", kind="attention", batch=1, longest=500, most=1, page=16, heads=32, kv_heads=32, d=128, dtype="bf16",
             cap=0.0, window=0, slopes=False, heads_first=False),
        # an ordinary decode step, requests of all lengths
        dict(name="attention_decode", kind="attention", batch=64, longest=4096, most=1, page=16, heads=32, kv_heads=8, d=128, dtype="bf16",
             cap=0.0, window=0, slopes=False, heads_first=False),
        # few requests over long documents, capped scores
        dict(name="attention_long", kind="attention", batch=4, longest=131072, most=1, page=64, heads=32, kv_heads=8, d=128, dtype="f16",
             cap=30.0, window=0, slopes=False, heads_first=True),
        # a chunk of two prompts behind what is cached of them
        dict(name="attention_chunk", kind="attention", batch=2, longest=6000, most=1000, page=16, heads=32, kv_heads=8, d=128, dtype="bf16",
             cap=0.0, window=0, slopes=False, heads_first=False),
        # one token through a 4096 x 4096 layer: latency
        dict(name="linear_token", kind="linear", m=1, n=4096, k=4096, group=128, zero=False, dtype="bf16"),
        # sixteen requests through the benchmark's layer
        dict(name="linear_batch", kind="linear", m=16, n=11008, k=4096, group=128, zero=True, dtype="f16"),
        # more requests, and its way back
        dict(name="linear_back", kind="linear", m=61, n=4096, k=11008, group=64, zero=False, dtype="bf16"),
    ]


def _size(rng, lo, hi, step=1):
    """Log-uniform in [lo, hi], a multiple of `step`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(step, min(hi, max(lo, v)) // step * step)


def _draw(rng):
    kind = rng.choice(["pages", "cache", "attention", "attention", "attention", "linear", "linear"])
    if kind == "pages":
        return dict(kind=kind, batch=_size(rng, 1, 512), longest=_size(rng, 1, 4096), most=rng.choice([1, 1, 5, _size(rng, 8, 700)]),
                    page=rng.choice([16, 32, 64]))
    if kind == "cache":
        return dict(kind=kind, batch=_size(rng, 1, 128), longest=_size(rng, 1, 2048), most=rng.choice([1, 1, 4, _size(rng, 8, 2048)]),
                    page=rng.choice([16, 32, 64]), heads=rng.choice([1, 2, 4, 8, 12, 32]), d=rng.choice([64, 96, 128, 256]),
                    dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), heads_first=rng.random() < 0.5)
    if kind == "attention":
        heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 8), (16, 2), (28, 4), (8, 1), (12, 12), (40, 8), (8, 4)])
        longest = _size(rng, 1, 131072)
        return dict(kind=kind, batch=min(_size(rng, 1, 256), max(1, 524288 // longest)), longest=longest,
                    most=rng.choice([1, 1, 1, rng.randint(2, 8), _size(rng, 8, 1000)]), page=rng.choice([16, 32, 64]), heads=heads,
                    kv_heads=kv_heads, d=rng.choice([64, 96, 128, 128, 128, 256]), dtype=rng.choice(["bf16", "f16"]),
                    cap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, 0, 1000]), slopes=rng.random() < 0.25,
                    heads_first=rng.random() < 0.5)
    group = rng.choice([32, 64, 128])
    step = rng.choice([64, 64, 1])
    return dict(kind=kind, m=_size(rng, 1, 64), n=_size(rng, 500, 11008, step), k=_size(rng, 512, 11008, group), group=group,
                zero=rng.random() < 0.5, dtype=rng.choice(["bf16", "f16"]))


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        for what in ("bytes", "flops"):
            limits[c["kind"], what] = max(limits.get((c["kind"], what), 0), w[what])
    while True:
        case = _draw(rng)
        w = work(case)
        # (keys and values of the widest heads, and the scores of a chunk, as the plain form holds them)
        held = case["batch"] * case["longest"] * case["kv_heads"] * case["d"] if case["kind"] == "attention" else 0
        scores = case["batch"] * case["longest"] * case["most"] * case["heads"] if case["kind"] == "attention" else 0
        if all(w[what] <= limits[case["kind"], what] for what in ("bytes", "flops")) and held <= 1 << 30 and scores <= 1 << 30:
            if 3072 not in case.values():
                return case


def _lengths(case):
    """(tokens cached before the step, new tokens) of each request: few long ones, many short."""
    before, added = [], []
    for i in range(case["batch"]):
        f = (i + 1) / case["batch"]
        total = max(1, round(case["longest"] * f * f))
        new = min(total, max(1, round(case["most"] * f)))
        before.append(total - new)
        added.append(new)
    return before, added


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _encode(x):
    """[pages, page, heads, d] values as e4m3 and a power of two per page and head."""
    top = x.abs().amax(dim=(1, 3)).float()
    mantissa, exponent = torch.frexp(top)
    scale = torch.ldexp(torch.ones_like(top), exponent - 9 + (mantissa > 0.875))
    return (x / scale[:, None, :, None].to(x.dtype)).to(torch.float8_e4m3fn), scale


def _physical(x, heads_first):
    """[pages, page, heads, d], lying in memory in that order or head by head."""
    return x.transpose(1, 2).contiguous().transpose(1, 2) if heads_first else x


def _paged(case, gen):
    before, added = _lengths(case)
    order = torch.randperm(case["batch"], generator=gen, device="cuda").tolist()
    before, added = [before[i] for i in order], [added[i] for i in order]
    page = case["page"]
    width = -(-max(b + a for b, a in zip(before, added)) // page)
    held = [-(-(b + a) // page) for b, a in zip(before, added)]
    total = sum(held)
    pages = torch.randperm(total + 8, generator=gen, device="cuda").to(torch.int32)
    return before, added, held, width, pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["kind"]
    s = dict(case)
    if kind == "linear":
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        s["x"] = torch.randn((m, k), generator=gen, device="cuda").to(_DTYPE[case["dtype"]])
        s["w"] = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda", dtype=torch.uint8)
        s["scale"] = (torch.rand((n, k // group), generator=gen, device="cuda") * 0.01 + 0.002).to(_DTYPE[case["dtype"]])
        s["zeros"] = torch.randint(4, 12, (n, k // group), generator=gen, device="cuda", dtype=torch.uint8) if case["zero"] else None
        return s
    before, added, held, width, pages = _paged(case, gen)
    page, batch = case["page"], case["batch"]
    s["tokens"] = sum(added)
    if kind == "pages":
        # what the requests hold before the step; the free pages follow, in the order in which they are handed out
        table, at = torch.full((batch, width), -1, dtype=torch.int32), 0
        mine = pages.cpu()
        for b in range(batch):
            n = -(-before[b] // page)
            table[b, :n] = mine[at:at + n]
            at += n
        s.update(lengths=_ints(before), added=_ints(added), table=table.cuda(), free=pages[at:].contiguous())
        return s
    table, at, mine = torch.full((batch, width), -1, dtype=torch.int32), 0, pages.cpu()
    for b in range(batch):
        table[b, :held[b]] = mine[at:at + held[b]]
        at += held[b]
    count = pages.numel()
    if kind == "cache":
        shape = (count, page, case["heads"], case["d"])
        for name in ("k", "v"):
            # what is cached is a little smaller than what comes, so that some pages need a larger scale
            old = torch.randn(shape, generator=gen, device="cuda") * torch.rand((count, 1, case["heads"], 1), generator=gen, device="cuda")
            cache, s[name + "_scale"] = _encode(old)
            s[name + "_cache"] = _physical(cache.view(torch.uint8), case["heads_first"]).view(torch.float8_e4m3fn)
            s[name] = torch.randn((s["tokens"], case["heads"], case["d"]), generator=gen, device="cuda").to(_DTYPE[case["dtype"]])
        slots, touched = [], []
        rows = table.tolist()
        for b in range(batch):
            for p in range(before[b], before[b] + added[b]):
                slots.append(rows[b][p // page] * page + p % page)
            for c in range(before[b] // page, -(-(before[b] + added[b]) // page)):
                filled = min(page, before[b] + added[b] - c * page)
                touched += [rows[b][c] * page + i for i in range(filled)]
        s["slots"], s["touched"] = _ints(slots, torch.int64), _ints(touched, torch.int64)
        return s
    shape = (count, page, case["kv_heads"], case["d"])
    for name in ("k", "v"):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float16)
        x *= torch.rand((count, 1, case["kv_heads"], 1), generator=gen, device="cuda", dtype=torch.float16) + 0.5
        cache, s[name + "_scale"] = _encode(x)
        s[name + "_cache"] = _physical(cache.view(torch.uint8), case["heads_first"]).view(torch.float8_e4m3fn)
        del x, cache
    starts = [0]
    for a in added:
        starts.append(starts[-1] + a)
    s["q"] = torch.randn((s["tokens"], case["heads"], case["d"]), generator=gen, device="cuda").to(_DTYPE[case["dtype"]])
    s["table"], s["lengths"] = table.cuda(), _ints([b + a for b, a in zip(before, added)])
    s["starts"] = _ints(starts) if case["most"] > 1 else None
    # 2^(-8 h / heads): the nearer heads forget sooner
    s["bias"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["heads"]) for h in range(case["heads"])], device="cuda") if case["slopes"] else None
    return s


def run(s):
    return (_own if own else _plain)[s["kind"]](s)


# ---- the framework's operators ----

def _own_pages(s):
    from kernelcodegen_amd import ops
    slots, positions, starts, lengths, used = ops.page_slots(s["lengths"], s["added"], s["table"], s["free"], s["page"], s["tokens"])
    return dict(slots=slots, positions=positions, starts=starts, lengths=lengths, used=used, table=s["table"])


def _own_cache(s):
    from kernelcodegen_amd import ops
    ops.cache_write(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"])
    dtype = _DTYPE[s["dtype"]]
    return dict(k=ops.cache_read(s["k_cache"], s["k_scale"], s["touched"], dtype), k_scale=s["k_scale"],
                v=ops.cache_read(s["v_cache"], s["v_scale"], s["touched"], dtype), v_scale=s["v_scale"])


def _own_attention(s):
    from kernelcodegen_amd import ops
    return ops.cache_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"], s["lengths"], starts=s["starts"],
                               cap=s["cap"] or None, window=s["window"] or None, slopes=s["bias"])


def _own_linear(s):
    from kernelcodegen_amd import ops
    return ops.matmul_q4(s["x"], s["w"], s["scale"], zero=s["zeros"])


# ---- the same in elementary operations ----

def _plain_pages(s):
    lengths, added, table, free, page = s["lengths"], s["added"], s["table"], s["free"], s["page"]
    device, count, width = lengths.device, free.numel(), table.shape[1]
    before, after = (lengths + page - 1) // page, (lengths + added + page - 1) // page
    need = after - before
    first = torch.cumsum(need, 0, dtype=torch.int32) - need
    column = torch.arange(width, dtype=torch.int32, device=device)[None, :]
    at = first[:, None] + column - before[:, None]
    new = (column >= before[:, None]) & (column < after[:, None])
    got = new & (at < count)
    table[:] = torch.where(got, free[at.clamp(0, count - 1).long()], table)
    starts = torch.zeros(lengths.numel() + 1, dtype=torch.int32, device=device)
    starts[1:] = torch.cumsum(added, 0, dtype=torch.int32)
    token = torch.arange(s["tokens"], dtype=torch.int32, device=device)
    request = torch.searchsorted(starts[1:].contiguous(), token, right=True).clamp(max=lengths.numel() - 1)
    real = token < starts[-1]
    position = torch.where(real, lengths[request] + token - starts[request], -1)
    of = (position // page).clamp(0, width - 1).long()
    entry = torch.where((new & ~got)[request, of], -1, table[request, of])
    fits = real & (position // page < width) & (entry >= 0)
    slots = torch.where(fits, entry.long() * page + (position % page).long(), -1)
    return dict(slots=slots, positions=position, starts=starts, lengths=lengths + added, used=need.sum(dtype=torch.int32).clamp(max=count).reshape(1),
                table=table)


def _power(top):
    """The least power of two whose 448-fold reaches `top`; 0 for 0."""
    mantissa, exponent = torch.frexp(top)
    power = torch.ldexp(torch.ones_like(top), torch.clamp(exponent - 9 + (mantissa > 0.875), min=-126))
    return torch.where(top > 0, power, 0.0)


def _plain_write(x, cache, scale, slots, page):
    pages, heads = scale.shape
    at, row = slots // page, slots % page
    x = x.float()
    top = torch.zeros_like(scale).scatter_reduce(0, at[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    first = torch.full((pages,), page, dtype=torch.int64, device=x.device).scatter_reduce(0, at, row, "amin")
    touched = (first < page).nonzero()[:, 0]
    need, old = _power(top[touched]), scale[touched]
    now = torch.where(first[touched, None] > 0, torch.maximum(old, need), need)
    held = cache[touched].float() * torch.where(now > 0, old / now, 0.0)[:, None, :, None]
    keep = torch.arange(page, device=x.device)[None, :] < first[touched, None]
    raw = cache.view(torch.uint8)
    raw[touched] = torch.where(keep[:, :, None, None], held.to(torch.float8_e4m3fn).view(torch.uint8), raw[touched])
    scale[touched] = now
    mine = scale[at][:, :, None]
    raw[at, row] = torch.where(mine > 0, x / mine, 0.0).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_read(cache, scale, slots, page, dtype):
    at = slots // page
    return (cache.view(torch.uint8)[at, slots % page].view(torch.float8_e4m3fn).float() * scale[at][:, :, None]).to(dtype)


def _plain_cache(s):
    _plain_write(s["k"], s["k_cache"], s["k_scale"], s["slots"], s["page"])
    _plain_write(s["v"], s["v_cache"], s["v_scale"], s["slots"], s["page"])
    dtype = _DTYPE[s["dtype"]]
    return dict(k=_plain_read(s["k_cache"], s["k_scale"], s["touched"], s["page"], dtype), k_scale=s["k_scale"],
                v=_plain_read(s["v_cache"], s["v_scale"], s["touched"], s["page"], dtype), v_scale=s["v_scale"])


def _gathered(cache, scale, table, page):
    """[batch, heads, keys, d] in fp32."""
    held = table.clamp(min=0).long()
    x = cache.view(torch.uint8)[held].view(torch.float8_e4m3fn).float() * scale[held][:, :, None, :, None]
    return x.flatten(1, 2).transpose(1, 2).contiguous()


def _plain_attention(s):
    q, table, lengths, page, most = s["q"], s["table"], s["lengths"], s["page"], s["most"]
    batch, heads, kv_heads, d = lengths.numel(), s["heads"], s["kv_heads"], s["d"]
    group, keys = heads // kv_heads, table.shape[1] * page
    starts = torch.arange(batch + 1, dtype=torch.int32, device=q.device) if s["starts"] is None else s["starts"]
    count = starts[1:] - starts[:-1]
    step = torch.arange(most, device=q.device)[None, :]
    row = (starts[:-1, None] + step).clamp(max=q.shape[0] - 1)
    real = step < count[:, None]
    position = lengths[:, None] - count[:, None] + step                                           # [batch, most]
    k, v = _gathered(s["k_cache"], s["k_scale"], table, page), _gathered(s["v_cache"], s["v_scale"], table, page)
    key = torch.arange(keys, device=q.device)
    v = torch.where((key[None, :] < lengths[:, None])[:, None, :, None], v, 0.0)
    x = q[row].float().view(batch, most, kv_heads, group, d).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * most, d)
    score = (x @ k.transpose(2, 3)).mul_(d ** -0.5).view(batch, kv_heads, group, most, keys)
    if s["cap"]:
        score = score.div_(s["cap"]).tanh_().mul_(s["cap"])
    distance = key[None, None, :] - position[:, :, None]                                          # [batch, most, keys]
    if s["bias"] is not None:
        score += s["bias"].view(1, kv_heads, group, 1, 1) * distance[:, None, None]
    seen = (distance <= 0) & real[:, :, None]
    if s["window"]:
        seen &= distance > -s["window"]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(batch, kv_heads, group * most, keys) @ v).view(batch, kv_heads, group, most, d) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, d)
    # rows in the order of q: those of a request lie together
    token = torch.arange(q.shape[0], device=q.device)
    request = torch.searchsorted(starts[1:].contiguous(), token.to(torch.int32), right=True).clamp(max=batch - 1)
    return out[request, (token - starts[request]).clamp(0, most - 1)].to(q.dtype)


def _plain_linear(s):
    w, n, k, group = s["w"], s["n"], s["k"], s["group"]
    q = torch.stack((w & 15, w >> 4), -1).view(n, k // group, group).float()
    q = (q - (8.0 if s["zeros"] is None else s["zeros"].float()[:, :, None])) * s["scale"].float()[:, :, None]
    return (s["x"].float() @ q.view(n, k).t()).to(s["x"].dtype)


_own = dict(pages=_own_pages, cache=_own_cache, attention=_own_attention, linear=_own_linear)
_plain = dict(pages=_plain_pages, cache=_plain_cache, attention=_plain_attention, linear=_plain_linear)


def work(case):
    kind = case["kind"]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        groups = n * (k // case["group"])
        return {"bytes": n * k // 2 + groups * (2 + (1 if case["zero"] else 0)) + 2 * m * (n + k), "flops": 2 * m * n * k}
    before, added = _lengths(case)
    page = case["page"]
    tokens = sum(added)
    if kind == "pages":
        taken = sum(-(-(b + a) // page) - -(-b // page) for b, a in zip(before, added))
        return {"bytes": 8 * case["batch"] + 8 * taken + 12 * tokens + 8 * case["batch"] + 8, "flops": 0}
    if kind == "cache":
        row = case["heads"] * case["d"]
        touched = sum(min(b + a, -(-(b + a) // page) * page) - b // page * page for b, a in zip(before, added))
        # new rows in and out in 8 bits, touched rows read and given in the cases' type; keys and values
        return {"bytes": 2 * row * (tokens * (_SIZE[case["dtype"]] + 1) + touched * (1 + _SIZE[case["dtype"]])) + 16 * (tokens + touched), "flops": 0}
    pairs, keys = 0, 0
    for b, a in zip(before, added):
        seen = [min(b + i + 1, case["window"] or b + i + 1) for i in range(a)]
        pairs += sum(seen)
        keys += min(b + a, (case["window"] or b + a) + a - 1)
    return {"bytes": 2 * keys * case["kv_heads"] * (case["d"] + 4 / page) + 4 * tokens * case["heads"] * case["d"],
            "flops": 4 * pairs * case["heads"] * case["d"]}


# ---- the definitions in 64 bits ----

def _exact_pages(s):
    page, width = s["page"], s["table"].shape[1]
    lengths, added, free = s["lengths"].tolist(), s["added"].tolist(), s["free"].tolist()
    table, slots, positions, starts, used = s["table"].tolist(), [], [], [0], 0
    for b in range(len(lengths)):
        for p in range(lengths[b], lengths[b] + added[b]):
            if p % page == 0:
                table[b][p // page] = free[used]
                used += 1
            positions.append(p)
            slots.append(table[b][p // page] * page + p % page)
        starts.append(starts[-1] + added[b])
    assert all(len(row) == width for row in table)
    return dict(slots=torch.tensor(slots), positions=torch.tensor(positions, dtype=torch.int32), starts=torch.tensor(starts, dtype=torch.int32),
                lengths=torch.tensor([x + y for x, y in zip(lengths, added)], dtype=torch.int32), used=torch.tensor([used], dtype=torch.int32),
                table=torch.tensor(table, dtype=torch.int32))


def _nearest_e4m3(x):
    """Values of the 8-bit format nearest to x (|x| <= 448), ties to the even one: steps of 2^(e-3), and of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_cache(s):
    page, out = s["page"], {}
    slots, touched = s["slots"], s["touched"]
    pages = slots // page
    # slots of a page lie together: where each page's run begins, and its first row
    lead = torch.ones_like(slots, dtype=torch.bool)
    lead[1:] = pages[1:] != pages[:-1]
    run = torch.cumsum(lead, 0) - 1
    at, first = pages[lead], (slots % page)[lead]
    for name in ("k", "v"):
        x, scale = s[name].double(), s[name + "_scale"].double()
        value = s[name + "_cache"].float().double()[at]
        top = x.abs().amax(-1)
        most = torch.zeros(at.numel(), top.shape[1], dtype=torch.float64, device=x.device).index_reduce(0, run, top, "amax")
        need = torch.exp2(torch.ceil(torch.log2(most / 448.0)))
        now = torch.where((first > 0)[:, None], torch.maximum(scale[at], need), need)
        held = _nearest_e4m3(value * (scale[at] / now)[:, None, :, None])
        held[run, slots % page] = _nearest_e4m3(x / now[run][:, :, None])
        scale = scale.clone()
        scale[at] = now
        of = torch.full((scale.shape[0],), -1, dtype=torch.int64, device=x.device)
        of[at] = torch.arange(at.numel(), device=x.device)
        out[name] = held[of[touched // page], touched % page] * scale[touched // page][:, :, None]
        out[name + "_scale"] = scale
    return out


def _exact_attention(s):
    d, page, group = s["d"], s["page"], s["heads"] // s["kv_heads"]
    lengths, rows = s["lengths"].tolist(), []
    starts = list(range(len(lengths) + 1)) if s["starts"] is None else s["starts"].tolist()
    for b, length in enumerate(lengths):
        held = s["table"][b, :-(-length // page)].long()
        k, v = ((s[n + "_cache"].view(torch.uint8)[held].view(torch.float8_e4m3fn).double() * s[n + "_scale"][held].double()[:, None, :, None])
                .reshape(-1, s["kv_heads"], d)[:length] for n in ("k", "v"))
        q = s["q"][starts[b]:starts[b + 1]].double()
        behind = torch.arange(length - q.shape[0], length, device=q.device)[:, None] - torch.arange(length, device=q.device)[None, :]
        hidden = (behind < 0) | (behind >= s["window"] if s["window"] else behind < 0)
        heads = []
        for h in range(s["heads"]):
            t = q[:, h] @ k[:, h // group].t() / math.sqrt(d)
            t = s["cap"] * torch.tanh(t / s["cap"]) if s["cap"] else t
            t = t - float(s["bias"][h]) * behind if s["bias"] is not None else t
            heads.append(torch.softmax(t.masked_fill(hidden, -math.inf), -1) @ v[:, h // group])
        rows.append(torch.stack(heads, 1))
    return torch.cat(rows)


def exact(case, seed):
    kind = case["kind"]
    w = work(case)
    if w["flops"] > 2e12 or (kind == "attention" and case["batch"] * case["heads"] > 12000):
        return None
    s = prepare(case, seed)
    if kind == "pages":
        return _exact_pages(s)
    if kind == "cache":
        return _exact_cache(s)
    if kind == "attention":
        return _exact_attention(s)
    scale = s["scale"].double().repeat_interleave(s["group"], 1)
    zero = 8 if s["zeros"] is None else s["zeros"].double().repeat_interleave(s["group"], 1)
    code = torch.empty(s["n"], s["k"], dtype=torch.float64, device="cuda")
    code[:, 0::2], code[:, 1::2] = s["w"].double() % 16, torch.div(s["w"], 16, rounding_mode="floor").double()
    return s["x"].double() @ (scale * (code - zero)).t()
