"""A small language model that answers several requests at once, from the operators of a decoding step: page tables and an 8-bit cache
of keys and values, attention over it, and products with 4-bit weights.

    python -m kernelcodegen_amd.decode [--requests 8] [--tokens 64] [--layers 4]

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


class Decoder:
    """Layers of attention (with a bias by distance, so that it needs no positions) and two products, for `batch` requests of up to
    `width` pages each, which share `pages` pages."""

    def __init__(self, batch, layers=4, heads=16, kv_heads=4, d=64, wide=4096, vocab=4096, group=64, page=16, pages=512, width=64, seed=0):
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

    def step(self, tokens, added=None):
        """Takes the new tokens of all requests, int64 [T], those of a request beside one another: added[b] (int32 [B]) of request b, or
        one of each.  Returns the scores of each request's next token, [B, vocab] (nothing of use for a request that gets none)."""
        rows = tokens.shape[0]
        slots, _, starts, lengths, used = ops.page_slots(self.lengths, self._one if added is None else added, self.table, self.free, self.page, rows)
        x = ops.gather(self.embedding, tokens).view(rows, -1)
        for layer in self.layers:
            (kc, ks), (vc, vs) = layer["keys"], layer["values"]
            qkv = ops.matmul_q4(ops.layernorm(x, *layer["norms"][0], 1), *layer["qkv"]).view(rows, -1, self.d)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            ops.cache_write(k, v, kc, vc, ks, vs, slots)
            seen = ops.cache_attention(q, kc, vc, ks, vs, self.table, lengths, starts=None if added is None else starts, slopes=self.slopes)
            x = ops.binary(x, ops.matmul_q4(seen.view(rows, -1), *layer["out"]), "Add")
            wide = ops.elementwise(ops.matmul_q4(ops.layernorm(x, *layer["norms"][1], 1), *layer["up"]), "Gelu")
            x = ops.binary(x, ops.matmul_q4(wide, *layer["down"]), "Add")
        self.lengths.copy_(lengths)
        left = self._order + used
        self.free.copy_(torch.where(left < len(self.free), self.free[left.clamp(max=len(self.free) - 1)], -1))
        if added is not None:
            x = ops.gather(x, (starts[1:] - 1).long()).view(len(self.lengths), -1)
        return ops.matmul_q4(ops.layernorm(x, *self.last, 1), *self.head)

    def record(self, tokens):
        """A HIP graph of a step of one token each, which takes `tokens` and leaves the likeliest next ones there; replay() is a step.
        A step has to have run before it, so that every kernel is loaded."""
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            tokens.copy_(self.step(tokens).argmax(-1))
        return graph


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--requests", type=int, default=8)
    parser.add_argument("--tokens", type=int, default=64)
    parser.add_argument("--layers", type=int, default=4)
    asked = parser.parse_args()
    if not (1 <= asked.requests <= 64 and 2 <= asked.tokens <= 512 and 1 <= asked.layers <= 64):
        parser.error("1 to 64 requests, 2 to 512 tokens, 1 to 64 layers")
    model = Decoder(asked.requests, layers=asked.layers, pages=asked.requests * 64)
    prompts = [17 + 31 * b % 400 for b in range(asked.requests)]
    scores = model.step(torch.randint(0, 4096, (sum(prompts),), device="cuda"), torch.tensor(prompts, device="cuda", dtype=torch.int32))
    tokens = scores.argmax(-1)
    tokens.copy_(model.step(tokens).argmax(-1))
    graph = model.record(tokens)
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


if __name__ == "__main__":
    main()
