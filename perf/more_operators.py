"""Performance cases of the operators around a decoding step: positions, adapters, and what an answer was worth.

    append    queries and keys rotated by their positions; keys and values written into the 8-bit cache on the way, and the rows of the
              pages that this touched read back
    adapters  low-rank adapters of many requests beside a shared projection, whose result they are added to
    logprobs  log probabilities of given tokens, entropies, and the likeliest alternatives with theirs

`own` False computes them in elementary torch operations, True through `kernelcodegen_amd.ops`.
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # one decode step of 64 requests: a token each; latency
        dict(name="append_decode", kind="append", batch=64, longest=2000, most=1, page=16, heads=32, kv_heads=8, d=128, rotated=128,
             interleaved=False, dtype="bf16", heads_first=False),
        # a few short answers of a small model in fp32, half of each head rotated by neighbours, pages head by head
        dict(name="append_small", kind="append", batch=3, longest=77, most=5, page=32, heads=12, kv_heads=12, d=64, rotated=32,
             interleaved=True, dtype="f32", heads_first=True),
        # prompts: whole pages at a time
        dict(name="append_prompts", kind="append", batch=9, longest=2048, most=2048, page=16, heads=32, kv_heads=8, d=128, rotated=128,
             interleaved=False, dtype="f16", heads_first=False),
        # one request with an adapter: latency
        dict(name="adapters_token", kind="adapters", batch=1, most=1, adapters=8, rank=16, n=4096, k=4096, dtype="bf16", out="bf16"),
        # a decode step of 64 requests with 40 adapters between them
        dict(name="adapters_decode", kind="adapters", batch=64, most=1, adapters=40, rank=16, n=4096, k=4096, dtype="bf16", out="bf16"),
        # prompts of a dozen requests through the benchmark's layer, its result in fp32
        dict(name="adapters_prompts", kind="adapters", batch=12, most=400, adapters=9, rank=32, n=11008, k=4096, dtype="f16", out="f32"),
        # one long batch of prompts with adapters of a high rank
        dict(name="adapters_long", kind="adapters", batch=4, most=2000, adapters=3, rank=64, n=4096, k=4096, dtype="bf16", out="bf16"),
        # the next token of one request, with a few alternatives: latency
        dict(name="logprobs_token", kind="logprobs", rows=1, vocab=32000, top=5, dtype="bf16"),
        # a decode step over a large vocabulary in fp32
        dict(name="logprobs_decode", kind="logprobs", rows=64, vocab=128000, top=20, dtype="f32"),
        # a vocabulary of an odd size, more rows than compute units
        dict(name="logprobs_odd", kind="logprobs", rows=500, vocab=50021, top=10, dtype="f16"),
        # a prompt is scored: every token of it, no alternatives
        dict(name="logprobs_prompt", kind="logprobs", rows=2000, vocab=32000, top=0, dtype="bf16"),
    ]


def _size(rng, lo, hi, step=1):
    """Log-uniform in [lo, hi], a multiple of `step`."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(step, min(hi, max(lo, v)) // step * step)


def _draw(rng):
    kind = rng.choice(["append", "adapters", "adapters", "logprobs", "logprobs"])
    if kind == "append":
        heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 8), (16, 2), (28, 4), (8, 1), (12, 12), (40, 8)])
        d = rng.choice([64, 96, 128, 128, 256])
        return dict(kind=kind, batch=_size(rng, 1, 128), longest=_size(rng, 1, 2048), most=rng.choice([1, 1, 4, _size(rng, 8, 2048)]),
                    page=rng.choice([16, 32, 64]), heads=heads, kv_heads=kv_heads, d=d, rotated=rng.choice([d, d, d // 2]),
                    interleaved=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), heads_first=rng.random() < 0.5)
    if kind == "adapters":
        step = rng.choice([64, 64, 8])
        return dict(kind=kind, batch=_size(rng, 1, 128), most=rng.choice([1, 1, 1, 4, _size(rng, 8, 2000)]), adapters=_size(rng, 1, 64),
                    rank=rng.choice([8, 16, 16, 32, 64]), n=_size(rng, 500, 11008, rng.choice([step, 1])), k=_size(rng, 512, 11008, step),
                    dtype=rng.choice(["bf16", "f16"]), out=rng.choice(["same", "same", "f32"]))
    return dict(kind=kind, rows=_size(rng, 1, 2000), vocab=_size(rng, 1000, 260000, rng.choice([64, 1])), top=rng.choice([0, 1, 5, 10, 20]),
                dtype=rng.choice(["bf16", "f16", "f32"]))


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        for what in ("bytes", "flops"):
            limits[c["kind"], what] = max(limits.get((c["kind"], what), 0), w[what])
    while True:
        case = _draw(rng)
        if case.get("out") == "same":
            case["out"] = case["dtype"]
        w = work(case)
        if all(w[what] <= limits[case["kind"], what] for what in ("bytes", "flops")):
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


def _counts(case):
    """New tokens of each request."""
    return [max(1, round(case["most"] * (i + 1) / case["batch"])) for i in range(case["batch"])]


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _two(n):
    """2^n in 32 bits, n from -126 on, put together from bits (a power function need not be exact)."""
    return (n.to(torch.int32) + 127 << 23).view(torch.float32)


def _encode(x):
    """[pages, page, heads, d] values as e4m3 and a power of two per page and head."""
    top = x.abs().amax(dim=(1, 3)).float()
    mantissa, exponent = torch.frexp(top)
    scale = _two(exponent - 9 + (mantissa > 0.875))
    return (x / scale[:, None, :, None].to(x.dtype)).to(torch.float8_e4m3fn), scale


def _prepare_append(s, gen):
    before, added = _lengths(s)
    order = torch.randperm(s["batch"], generator=gen, device="cuda").tolist()
    before, added = [before[i] for i in order], [added[i] for i in order]
    page, d, dtype = s["page"], s["d"], _DTYPE[s["dtype"]]
    held = [-(-(b + a) // page) for b, a in zip(before, added)]
    count, tokens = sum(held) + 8, sum(added)
    mine, at = torch.randperm(count, generator=gen, device="cuda").tolist(), 0
    slots, touched, positions = [], [], []
    for b, a, n in zip(before, added, held):
        row, at = mine[at:at + n], at + n
        for p in range(b, b + a):
            slots.append(row[p // page] * page + p % page)
            positions.append(p)
        for c in range(b // page, n):
            touched += [row[c] * page + i for i in range(min(page, b + a - c * page))]
    for name in ("k", "v"):
        # what is cached is a little smaller than what comes, so that some pages need a larger scale
        old = torch.randn((count, page, s["kv_heads"], d), generator=gen, device="cuda")
        old *= torch.rand((count, 1, s["kv_heads"], 1), generator=gen, device="cuda")
        cache, s[name + "_scale"] = _encode(old)
        raw = cache.view(torch.uint8)
        s[name + "_cache"] = (raw.transpose(1, 2).contiguous().transpose(1, 2) if s["heads_first"] else raw).view(torch.float8_e4m3fn)
    # one projection gives all three
    heads = (s["heads"], s["kv_heads"], s["kv_heads"])
    qkv = torch.randn((tokens, sum(heads), d), generator=gen, device="cuda").to(dtype)
    s["q"], s["k"], s["v"] = qkv.split(heads, 1)
    s["slots"], s["positions"], s["touched"] = _ints(slots, torch.int64), _ints(positions), _ints(touched, torch.int64)
    rate = 10000.0 ** (-torch.arange(s["rotated"] // 2, dtype=torch.float64, device="cuda") * 2 / s["rotated"])
    angle = torch.arange(max(s["longest"], 1), dtype=torch.float64, device="cuda")[:, None] * rate[None, :]
    s["rotation"] = torch.cat((angle.cos(), angle.sin()), 1).float()


def _prepare_adapters(s, gen):
    counts, dtype, n, k, rank, adapters = _counts(s), _DTYPE[s["dtype"]], s["n"], s["k"], s["rank"], s["adapters"]
    order = torch.randperm(s["batch"], generator=gen, device="cuda").tolist()
    # adapters in turn, and every so often a request without one
    which = [min(i % (adapters + 1), adapters) for i in range(s["batch"])]
    names = torch.randperm(adapters, generator=gen, device="cuda").tolist() + [-1]
    tokens = sum(counts)
    s["which"] = _ints([names[which[i]] for i in order for _ in range(counts[i])])
    s["x"] = torch.randn((tokens, k), generator=gen, device="cuda").to(dtype)
    s["y"] = torch.randn((tokens, n), generator=gen, device="cuda").to(_DTYPE[s["out"]])
    s["a"] = (torch.randn((adapters, rank, k), generator=gen, device="cuda") * k ** -0.5).to(dtype)
    s["b"] = (torch.randn((adapters, n, rank), generator=gen, device="cuda") * 0.1).to(dtype)
    s["scale"] = torch.rand(adapters, generator=gen, device="cuda") * 1.75 + 0.25


def _prepare_logprobs(s, gen):
    rows, vocab = s["rows"], s["vocab"]
    logits = torch.randn((rows, vocab), generator=gen, device="cuda")
    logits *= torch.rand((rows, 1), generator=gen, device="cuda") * 4 + 1
    banned = torch.randperm(vocab - 1, generator=gen, device="cuda")[:vocab // 500] + 1
    logits[:, banned] = -math.inf
    s["logits"] = logits.to(_DTYPE[s["dtype"]])
    # half of the tokens are likely ones
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    likely = logits[:, :1000].argmax(1)
    tokens = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, likely, tokens)
    s["tokens"] = torch.where(torch.isin(tokens, banned), 0, tokens)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = dict(case)
    {"append": _prepare_append, "adapters": _prepare_adapters, "logprobs": _prepare_logprobs}[case["kind"]](s, gen)
    return s


def run(s):
    return (_own if own else _plain)[s["kind"]](s)


# ---- the framework's operators ----

def _own_append(s):
    from kernelcodegen_amd import ops
    q = ops.cache_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["slots"], s["positions"], s["rotation"],
                         interleaved=s["interleaved"])
    dtype = _DTYPE[s["dtype"]]
    return dict(q=q, k=ops.cache_read(s["k_cache"], s["k_scale"], s["touched"], dtype), k_scale=s["k_scale"],
                v=ops.cache_read(s["v_cache"], s["v_scale"], s["touched"], dtype), v_scale=s["v_scale"])


def _own_adapters(s):
    from kernelcodegen_amd import ops
    return ops.add_adapters(s["y"], s["x"], s["a"], s["b"], s["which"], scale=s["scale"])


def _own_logprobs(s):
    from kernelcodegen_amd import ops
    return ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])


# ---- the same in elementary operations ----

def _turn(x, s):
    """Rows [tokens, heads, d] turned by their positions, in 64 bits, since what becomes of a key in 8 bits jumps at borders."""
    r = s["rotated"]
    table = s["rotation"][s["positions"].long()].double()[:, None, :]
    c, w = table[..., :r // 2], table[..., r // 2:]
    x = x.double()
    if s["interleaved"]:
        one, two = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((one * c - two * w, two * c + one * w), -1).flatten(-2)
    else:
        one, two = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat((one * c - two * w, two * c + one * w), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _power(top):
    """The least power of two whose 448-fold reaches `top`; 0 for 0."""
    mantissa, exponent = torch.frexp(top)
    power = _two(torch.clamp(exponent - 9 + (mantissa > 0.875), min=-126))
    return torch.where(top > 0, power, 0.0)


def _bits(x):
    """Numbers in 64 bits (|x| <= 448) as the nearest of the 8-bit format: four binary digits, or a multiple of 2^-9."""
    step = _two(torch.clamp(torch.frexp(x)[1] - 4, min=-9)).double()
    return (torch.round(x / step) * step).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_write(x, cache, scale, slots, page):
    pages, heads = scale.shape
    at, row = slots // page, slots % page
    top = torch.zeros((pages, heads), dtype=x.dtype, device=x.device).scatter_reduce(0, at[:, None].expand(-1, heads), x.abs().amax(-1), "amax")
    first = torch.full((pages,), page, dtype=torch.int64, device=x.device).scatter_reduce(0, at, row, "amin")
    touched = (first < page).nonzero()[:, 0]
    need, old = _power(top[touched]), scale[touched]
    now = torch.where(first[touched, None] > 0, torch.maximum(old, need), need)
    held = cache[touched].float() * torch.where(now > 0, old / now, 0.0)[:, None, :, None]
    keep = torch.arange(page, device=x.device)[None, :] < first[touched, None]
    raw = cache.view(torch.uint8)
    raw[touched] = torch.where(keep[:, :, None, None], held.to(torch.float8_e4m3fn).view(torch.uint8), raw[touched])
    scale[touched] = now
    mine = scale[at][:, :, None].double()
    raw[at, row] = _bits(torch.where(mine > 0, x / mine, 0.0))


def _plain_read(cache, scale, slots, page, dtype):
    at = slots // page
    return (cache.view(torch.uint8)[at, slots % page].view(torch.float8_e4m3fn).float() * scale[at][:, :, None]).to(dtype)


def _plain_append(s):
    dtype, page = _DTYPE[s["dtype"]], s["page"]
    q = _turn(s["q"], s).to(dtype)
    _plain_write(_turn(s["k"], s), s["k_cache"], s["k_scale"], s["slots"], page)
    _plain_write(s["v"].double(), s["v_cache"], s["v_scale"], s["slots"], page)
    return dict(q=q, k=_plain_read(s["k_cache"], s["k_scale"], s["touched"], page, dtype), k_scale=s["k_scale"],
                v=_plain_read(s["v_cache"], s["v_scale"], s["touched"], page, dtype), v_scale=s["v_scale"])


def _plain_adapters(s):
    x, y, which = s["x"].float(), s["y"].to(torch.float32, copy=True), s["which"].long()
    if x.shape[0] <= 128:
        # each token's own matrices
        of = which.clamp(min=0)
        h = torch.bmm(s["a"][of].float(), x[:, :, None])
        delta = torch.bmm(s["b"][of].float(), h)[:, :, 0] * s["scale"][of][:, None]
        return (y + torch.where(which[:, None] >= 0, delta, 0.0)).to(s["y"].dtype)
    for r in range(s["adapters"]):
        rows = (which == r).nonzero()[:, 0]
        y[rows] += (x[rows] @ s["a"][r].float().t()) @ s["b"][r].float().t() * s["scale"][r]
    return y.to(s["y"].dtype)


def _plain_logprobs(s):
    x, top = s["logits"].float(), s["top"]
    m = x.amax(-1, keepdim=True)
    d = x - m
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    entropy = total.log()[:, 0] - torch.where(e > 0, d * e, 0.0).sum(-1) / total[:, 0]
    logprob = (d.gather(1, s["tokens"][:, None]) - total.log())[:, 0]
    if top == 0:
        none = torch.empty((x.shape[0], 0), device=x.device)
        return logprob, entropy, none, none.long()
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    return logprob, entropy, d.gather(1, order) - total.log(), order


_own = dict(append=_own_append, adapters=_own_adapters, logprobs=_own_logprobs)
_plain = dict(append=_plain_append, adapters=_plain_adapters, logprobs=_plain_logprobs)


def work(case):
    kind = case["kind"]
    if kind == "append":
        before, added = _lengths(case)
        page, size, row, tokens = case["page"], _SIZE[case["dtype"]], case["kv_heads"] * case["d"], sum(added)
        touched = sum(b + a - b // page * page for b, a in zip(before, added))
        positions = len({p for b, a in zip(before, added) for p in range(b, b + a)})
        # queries in and out, new rows in and out in 8 bits, touched rows read and given in the case's type; the table's rows; slots and positions
        return {"bytes": 2 * tokens * case["heads"] * case["d"] * size + 2 * row * (tokens * (size + 1) + touched * (1 + size)) +
                positions * case["rotated"] * 4 + 12 * tokens + 16 * touched,
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["rotated"]}
    if kind == "adapters":
        counts, turn = _counts(case), case["adapters"] + 1
        used = min(case["batch"], case["adapters"])
        tokens, with_one = sum(counts), sum(c for i, c in enumerate(counts) if i % turn != case["adapters"])
        weights = used * case["rank"] * (case["n"] + case["k"])
        return {"bytes": 2 * weights + 2 * with_one * case["k"] + 2 * tokens * case["n"] * _SIZE[case["out"]] + 4 * tokens,
                "flops": 2 * with_one * case["rank"] * (case["n"] + case["k"])}
    return {"bytes": case["rows"] * (case["vocab"] * _SIZE[case["dtype"]] + 16 + 12 * case["top"]), "flops": 6 * case["rows"] * case["vocab"]}


# ---- the definitions in 64 bits ----

def _nearest_e4m3(x):
    """Values of the 8-bit format nearest to x (|x| <= 448), ties to the even one: steps of 2^(e-3), and of 2^-9 below 2^-6."""
    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    page, r, out = s["page"], s["rotated"], {}
    slots, touched = s["slots"], s["touched"]
    # a pair as a complex number, times that of its angle
    i = torch.arange(r // 2, device="cuda")
    first, second = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + r // 2)
    by = s["rotation"].double()[s["positions"].long()]
    by = torch.complex(by[:, i], by[:, i + r // 2])[:, None, :]
    new = {"v": s["v"].double()}
    for name in ("q", "k"):
        x = s[name].double()
        turned = torch.complex(x[..., first], x[..., second]) * by
        new[name] = x.clone()
        new[name][..., first], new[name][..., second] = turned.real, turned.imag
    out["q"] = new["q"]
    pages = slots // page
    # slots of a page lie together: where each page's run begins, and its first row
    lead = torch.ones_like(slots, dtype=torch.bool)
    lead[1:] = pages[1:] != pages[:-1]
    run_of = torch.cumsum(lead, 0) - 1
    at, begins = pages[lead], (slots % page)[lead]
    for name in ("k", "v"):
        x, scale = new[name], s[name + "_scale"].double()
        value = s[name + "_cache"].float().double()[at]
        top = x.abs().amax(-1)
        most = torch.zeros(at.numel(), top.shape[1], dtype=torch.float64, device=x.device).index_reduce(0, run_of, top, "amax")
        need = torch.exp2(torch.ceil(torch.log2(most / 448.0)))
        now = torch.where((begins > 0)[:, None], torch.maximum(scale[at], need), need)
        held = _nearest_e4m3(value * (scale[at] / now)[:, None, :, None])
        held[run_of, slots % page] = _nearest_e4m3(x / now[run_of][:, :, None])
        scale = scale.clone()
        scale[at] = now
        of = torch.full((scale.shape[0],), -1, dtype=torch.int64, device=x.device)
        of[at] = torch.arange(at.numel(), device=x.device)
        out[name] = held[of[touched // page], touched % page] * scale[touched // page][:, :, None]
        out[name + "_scale"] = scale
    return out


def _exact_adapters(s):
    out, which = s["y"].double(), s["which"]
    for r in sorted(set(which.tolist()) - {-1}):
        mine = which == r
        product = s["b"][r].double() @ s["a"][r].double() if int(mine.sum()) > 1000 else None
        x = s["x"][mine].double()
        delta = x @ product.t() if product is not None else torch.linalg.multi_dot((x, s["a"][r].double().t(), s["b"][r].double().t()))
        out[mine] += float(s["scale"][r]) * delta
    return out


def _exact_logprobs(s):
    parts = []
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        x = x.double()
        p = torch.log_softmax(x, -1)
        entropy = torch.special.entr(p.exp()).sum(-1)
        value, index = torch.sort(x, dim=-1, descending=True, stable=True) if s["top"] else (x, t[:, None])
        index = index[:, :s["top"]]
        parts.append((p.gather(1, t[:, None])[:, 0], entropy, p.gather(1, index), index))
    return tuple(torch.cat(p) for p in zip(*parts))


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "adapters": _exact_adapters, "logprobs": _exact_logprobs}[case["kind"]](s)
