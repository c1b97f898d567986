"""A small language model that answers several requests at once, from the operators of a decoding step: page tables and an 8-bit cache
of keys and values, attention over it, products with 4-bit weights, adapters of the requests' own beside them, and what an answer's tokens
were worth.

    python -m kernelcodegen_amd.decode [--requests 8] [--tokens 64] [--layers 4] [--rotated 64] [--adapters 3] [--top 2]

The weights are random; what it shows is how the operators go together.  One step takes the new tokens of all requests, whole prompts or
one token each; its work is on the device alone, so that the step of one token each is recorded once as a HIP graph and replayed for
every further token."""
import argparse
import time

import torch

from . import ops


def quantize_q4(w, group):
    """Rows of a matrix [N, K] as 4-bit codes with a scale and a zero for each `group` of a row: what ops.matmul_q4 takes."""
    n, k = w.shape
    parts = w.float().view(n, k // group, group)
    low, high = parts.amin(-1).clamp(max=0.0), parts.amax(-1).clamp(min=0.0)
    scale = ((high - low) / 15).clamp(min=1e-8).to(w.dtype)
    zero = (-low / scale.float()).round().clamp(0, 15)
    codes = ((parts / scale.float()[..., None]).round() + zero[..., None]).clamp(0, 15).to(torch.uint8).view(n, k)
    return (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous(), scale, zero.to(torch.uint8)


def rotations(positions, rotated, base=10000.0):
    """What ops.cache_append turns by: for each position the cosines of its `rotated` / 2 angles, then the sines.  Angles of far positions have
    more digits than fp32 holds, so they are taken in 64 bits."""
    rates = base ** (torch.arange(rotated // 2, dtype=torch.float64) * (-2 / rotated))
    angles = torch.arange(positions, dtype=torch.float64)[:, None] * rates
    return torch.cat((angles.cos(), angles.sin()), 1).float().cuda()


class Decoder:
    """Layers of attention and two products, for `batch` requests of up to `width` pages each, which share `pages` pages.  Attention has a bias by distance,
    and needs no positions, or queries and keys whose first `rotated` numbers are turned by them.  Beside the products around attention
    there are `adapters` adapters of a rank, of which each request may name one."""

    def __init__(self, batch, layers=4, heads=16, kv_heads=4, d=64, wide=4096, vocab=4096, group=64, page=16, pages=512, width=64, seed=0, rotated=0,
                 adapters=0, rank=16):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n, self.heads, self.kv_heads, self.d, self.page = heads * d, heads, kv_heads, d, page

        def product(rows, columns):
            return quantize_q4(torch.randn((rows, columns), generator=g, device="cuda").mul_(columns ** -0.5).half(), group)

        def norm():
            return torch.ones(n, device="cuda", dtype=torch.half), torch.zeros(n, device="cuda", dtype=torch.half)

        def cache():
            return (torch.zeros((pages, page, kv_heads, d), device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn),
                    torch.zeros((pages, kv_heads), device="cuda"))

        self.embedding = torch.randn((vocab, n), generator=g, device="cuda").half()
        self.layers = [dict(norms=(norm(), norm()), qkv=product((heads + 2 * kv_heads) * d, n), out=product(n, n), up=product(wide, n),
                            down=product(n, wide), keys=cache(), values=cache()) for _ in range(layers)]
        self.last, self.head = norm(), product(vocab, n)
        self.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")
        # on the device for good: what the requests have in the cache, their pages, and the free ones (-1 behind the last)
        self.lengths = torch.zeros(batch, device="cuda", dtype=torch.int32)
        self.table = torch.full((batch, width), -1, device="cuda", dtype=torch.int32)
        self.free = torch.arange(pages, device="cuda", dtype=torch.int32)
        self._order = torch.arange(pages, device="cuda")
        self._one = torch.ones(batch, device="cuda", dtype=torch.int32)
        self.rotation = rotations(width * page, rotated) if rotated else None

        def pool(rows, columns):
            return ((torch.randn((adapters, rank, columns), generator=g, device="cuda") * columns ** -0.5).half(),
                    (torch.randn((adapters, rows, rank), generator=g, device="cuda") * (0.5 * rank ** -0.5)).half())

        for layer in self.layers if adapters else ():
            layer["adapters"] = dict(qkv=pool((heads + 2 * kv_heads) * d, n), out=pool(n, n))

    def _product(self, layer, name, x, which):
        y = ops.matmul_q4(x, *layer[name])
        return y if which is None else ops.add_adapters(y, x, *layer["adapters"][name], which, inplace=True)

    def step(self, tokens, added=None, which=None):
        """Takes the new tokens of all requests, int64 [T], those of a request beside one another: added[b] (int32 [B]) of request b, or
        one of each; which: int32 [B], the adapter of each request (-1: none), the same in all its steps.  Returns the scores of each
        request's next token, [B, vocab] (nothing of use for a request that gets none)."""
        rows = tokens.shape[0]
        slots, positions, starts, lengths, used = ops.page_slots(self.lengths, self._one if added is None else added, self.table, self.free, self.page, rows)
        if which is not None and added is not None:
            which = which[torch.searchsorted(starts[1:], torch.arange(rows, device="cuda", dtype=torch.int32), right=True).clamp(max=len(which) - 1)]
        x = ops.gather(self.embedding, tokens).view(rows, -1)
        for layer in self.layers:
            (kc, ks), (vc, vs) = layer["keys"], layer["values"]
            qkv = self._product(layer, "qkv", ops.layernorm(x, *layer["norms"][0], 1), which).view(rows, -1, self.d)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            if self.rotation is None:
                ops.cache_write(k, v, kc, vc, ks, vs, slots)
            else:
                q = ops.cache_append(q, k, v, kc, vc, ks, vs, slots, positions, self.rotation)
            seen = ops.cache_attention(q, kc, vc, ks, vs, self.table, lengths, starts=None if added is None else starts,
                                       slopes=self.slopes if self.rotation is None else None)
            x = ops.binary(x, self._product(layer, "out", seen.view(rows, -1), which), "Add")
            wide = ops.elementwise(ops.matmul_q4(ops.layernorm(x, *layer["norms"][1], 1), *layer["up"]), "Gelu")
            x = ops.binary(x, ops.matmul_q4(wide, *layer["down"]), "Add")
        self.lengths.copy_(lengths)
        left = self._order + used
        self.free.copy_(torch.where(left < len(self.free), self.free[left.clamp(max=len(self.free) - 1)], -1))
        if added is not None:
            x = ops.gather(x, (starts[1:] - 1).long()).view(len(self.lengths), -1)
        return ops.matmul_q4(ops.layernorm(x, *self.last, 1), *self.head)

    def choose(self, scores, top=0):
        """The likeliest token of each row of scores, and what ops.token_logprobs gives for it: its log probability, the entropy, and those of `top`
        tokens with which they are."""
        tokens = scores.argmax(-1)
        return tokens, ops.token_logprobs(scores, tokens, top)

    def record(self, tokens, which=None, top=None):
        """A HIP graph of a step of one token each, which takes `tokens` and leaves the likeliest next ones there; replay() is a step.
        A step has to have run before it, so that every kernel is loaded.  With `top` it is given with the tensors where each step leaves
        what choose() tells."""
        graph, worth = torch.cuda.CUDAGraph(), None
        with torch.cuda.graph(graph):
            scores = self.step(tokens, which=which)
            if top is None:
                tokens.copy_(scores.argmax(-1))
            else:
                chosen, worth = self.choose(scores, top)
                tokens.copy_(chosen)
        return graph if top is None else (graph, worth)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--requests", type=int, default=8)
    parser.add_argument("--tokens", type=int, default=64)
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--rotated", type=int, default=0, help="numbers of a head that are turned by positions, a multiple of 16 up to 64; 0: a bias by distance")
    parser.add_argument("--adapters", type=int, default=0, help="adapters that the requests take in turn, one without each time")
    parser.add_argument("--top", type=int, default=0, help="alternatives to each token that are shown with their probabilities")
    asked = parser.parse_args()
    if not (1 <= asked.requests <= 64 and 2 <= asked.tokens <= 512 and 1 <= asked.layers <= 64):
        parser.error("1 to 64 requests, 2 to 512 tokens, 1 to 64 layers")
    if not (0 <= asked.rotated <= 64 and asked.rotated % 16 == 0 and 0 <= asked.adapters <= 64 and 0 <= asked.top <= 8):
        parser.error("0 to 64 rotated numbers, a multiple of 16, 0 to 64 adapters, 0 to 8 alternatives")
    model = Decoder(asked.requests, layers=asked.layers, pages=asked.requests * 64, rotated=asked.rotated, adapters=asked.adapters)
    which = torch.arange(asked.requests, device="cuda", dtype=torch.int32) % (asked.adapters + 1) - 1 if asked.adapters else None
    prompts = [17 + 31 * b % 400 for b in range(asked.requests)]
    scores = model.step(torch.randint(0, 4096, (sum(prompts),), device="cuda"), torch.tensor(prompts, device="cuda", dtype=torch.int32), which)
    tokens = scores.argmax(-1)
    tokens.copy_(model.step(tokens, which=which).argmax(-1))
    if asked.top:
        model.choose(scores, asked.top)
        graph, worth = model.record(tokens, which, asked.top)
    else:
        graph = model.record(tokens, which)
    answers = [tokens.clone()]
    torch.cuda.synchronize()
    begun = time.perf_counter()
    for _ in range(asked.tokens - 1):
        graph.replay()
        answers.append(tokens.clone())
    torch.cuda.synchronize()
    each = (time.perf_counter() - begun) / (asked.tokens - 1)
    print("prompts of %d tokens; then %.1f us a step, %.0f tokens/s" % (sum(prompts), each * 1e6, asked.requests / each))
    for b, answer in enumerate(torch.stack(answers, 1)[:8].tolist()):
        print("request %d: %s%s" % (b, " ".join(map(str, answer[:12])), " ..." if len(answer) > 12 else ""))
        if asked.top:
            logprob, entropy, best, names = worth
            print("  last token: probability %.3g, entropy %.2f; likeliest %s" % (
                logprob[b].exp(), entropy[b], ", ".join("%d (%.3g)" % (n, p) for n, p in zip(names[b].tolist(), best[b].exp().tolist()))))


if __name__ == "__main__":
    main()
