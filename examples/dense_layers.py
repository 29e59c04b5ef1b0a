"""The dense part of two layers of a hybrid model around the expert engine, run
as a server runs it: a prompt, then tokens one by one, for several streams.

    python examples/dense_layers.py [--streams 4] [--prompt 1024] [--tokens 64]

The first layer mixes tokens by the gated delta rule, whose state each stream
keeps in a row of a pool; the second by attention over the 8-bit paged cache. All
projections are 4-bit. Weights are random: what is shown is how the operators of
fronk_amd.dense go together (the experts' own calls would stand between the two
layers, on the same stream), and decoding replayed from a graph.
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from fronk_amd import dense  # noqa: E402


def quantize(w, group):
    """(codes, scales, zeros) of a matrix [rows, cols]: per group of a row the 16
    steps from its least to its largest value."""
    g = w.view(w.shape[0], -1, group)
    low, high = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
    scales = ((high - low) / 15).clamp(min=1e-4).to(torch.float16)
    zeros = torch.round(-low / scales.float()).clamp(0, 15)
    codes = (torch.round(g / scales.float()[..., None]) + zeros[..., None]).clamp(0, 15).to(torch.uint8).view(w.shape)
    return codes[:, 0::2] | codes[:, 1::2] << 4, scales, zeros.to(torch.uint8)


class Layers:
    def __init__(self, hidden=2560, key_heads=16, heads=32, key_dim=128, value_dim=128, q_heads=16, kv_heads=2, dim=256,
                 streams=4, context=4096, page=64, group=64, dtype=torch.bfloat16, seed=0):
        self.sizes = (key_heads, heads, key_dim, value_dim, q_heads, kv_heads, dim)
        self.dtype, self.page, self.streams = dtype, page, streams
        rand = torch.Generator(device="cuda").manual_seed(seed)

        def normal(*shape):
            return torch.randn(*shape, device="cuda", generator=rand)

        def weights(rows, cols):
            return quantize(normal(rows, cols) * cols ** -0.5, group)

        self.in1 = weights(2 * key_heads * key_dim + heads * value_dim, hidden)
        self.out1 = weights(hidden, heads * value_dim)
        self.in2 = weights((q_heads + 2 * kv_heads) * dim, hidden)
        self.out2 = weights(hidden, q_heads * dim)
        self.gates = normal(hidden, 2 * heads) * hidden ** -0.5
        self.rate = -torch.exp(normal(heads))
        # What a server keeps for its streams: states, the cache's pages and who has them.
        self.states = torch.zeros(streams, heads, key_dim, value_dim, device="cuda")
        per = (context + page - 1) // page
        self.cache = dense.KVCache.empty(streams * per, kv_heads, page, dim)
        self.table = torch.randperm(streams * per, device="cuda", generator=rand).to(torch.int32).view(streams, per)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def slots(self, stream, position):
        """Where tokens at these positions of these streams lie in the cache."""
        return self.table[stream, position // self.page] * self.page + (position % self.page).to(torch.int32)

    def forward(self, x, of, position, stream, offsets, longest, trace=None):
        """x [tokens, hidden] of sequences offsets [sequences + 1], at most
        `longest` tokens each; stream [sequences] is each one's row of the
        states, `of` [tokens] each token's stream, position [tokens] its place in
        it. `trace` takes the operators' operands."""
        key_heads, heads, dk, dv, q_heads, kv_heads, dim = self.sizes
        row = dense.q4_product(x, *self.in1)
        mixed = torch.nn.functional.silu(row)
        q = mixed[:, :key_heads * dk].unflatten(1, (key_heads, dk))
        k = mixed[:, key_heads * dk:2 * key_heads * dk].unflatten(1, (key_heads, dk))
        v = mixed[:, 2 * key_heads * dk:].unflatten(1, (heads, dv))
        gates = x.float() @ self.gates
        g = self.rate * torch.nn.functional.softplus(gates[:, :heads])
        beta = torch.sigmoid(gates[:, heads:])
        before = self.states.clone() if trace is not None else None
        o = dense.delta_rule(q, k, v, g, beta, self.states, self.states, offsets=offsets, slots=stream,
                             max_tokens=longest, normalize=True, status=self.status)
        h = x + dense.q4_product(o.flatten(1), *self.out1)

        row2 = dense.q4_product(h, *self.in2)
        q2 = row2[:, :q_heads * dim].unflatten(1, (q_heads, dim))
        k2 = row2[:, q_heads * dim:(q_heads + kv_heads) * dim].unflatten(1, (kv_heads, dim))
        v2 = row2[:, (q_heads + kv_heads) * dim:].unflatten(1, (kv_heads, dim))
        dense.kv_append(self.cache, k2, v2, self.slots(of, position), status=self.status)
        # Each token as a sequence of its own that ends with it.
        a = dense.kv_attend(self.cache, q2, self.table[of], (position + 1).to(torch.int32), status=self.status)
        y = h + dense.q4_product(a.flatten(1), *self.out2)
        if trace is not None:
            trace.update(row=row, q=q, k=k, v=v, g=g, beta=beta, before=before, o=o, h=h, row2=row2, q2=q2, a=a)
        return y


class Decoder:
    """One token of every stream, replayed from a graph: x in, y out. It keeps
    every tensor that the graph reads by its address."""

    def __init__(self, layers, length):
        n, hidden = layers.streams, layers.gates.shape[0]
        self.layers = layers
        self.x = torch.zeros(n, hidden, dtype=layers.dtype, device="cuda")
        self.of = torch.arange(n, device="cuda")
        self.position = torch.full((n,), length, dtype=torch.long, device="cuda")
        self.stream = torch.arange(n, dtype=torch.int32, device="cuda")
        self.offsets = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        kept = layers.states.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            self._token()
        torch.cuda.current_stream().wait_stream(side)
        layers.states.copy_(kept)   # (what the warm-up wrote to the cache, the first token overwrites)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph):
            self.y = self._token()
            self.position += 1

    def _token(self):
        return self.layers.forward(self.x, self.of, self.position, self.stream, self.offsets, 1)


def main():
    p = argparse.ArgumentParser()
    p.add_argument("--streams", type=int, default=4)
    p.add_argument("--prompt", type=int, default=1024)
    p.add_argument("--tokens", type=int, default=64)
    a = p.parse_args()
    layers = Layers(streams=a.streams, context=a.prompt + a.tokens)
    hidden = layers.gates.shape[0]
    x = torch.randn(a.streams * a.prompt, hidden, device="cuda").to(layers.dtype)
    stream = torch.arange(a.streams, dtype=torch.int32, device="cuda")
    of = torch.arange(a.streams, device="cuda").repeat_interleave(a.prompt)
    position = torch.arange(a.prompt, device="cuda").repeat(a.streams)
    offsets = torch.arange(a.streams + 1, dtype=torch.int32, device="cuda") * a.prompt
    for _ in range(2):   # the second time without the first call's loading
        layers.states.zero_()
        torch.cuda.synchronize()
        start = time.perf_counter()
        y = layers.forward(x, of, position, stream, offsets, a.prompt)
        torch.cuda.synchronize()
        prompt_ms = (time.perf_counter() - start) * 1e3
    decoder = Decoder(layers, a.prompt)
    decoder.x.copy_(y.view(a.streams, a.prompt, hidden)[:, -1])
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(a.tokens):
        decoder.graph.replay()
        decoder.x.copy_(decoder.y)
    torch.cuda.synchronize()
    ms = (time.perf_counter() - start) * 1e3 / a.tokens
    bad = layers.status.item()
    print(f"{a.streams} streams: prompts of {a.prompt} tokens {prompt_ms:.3f} ms, then {ms:.4f} ms a token each; "
          f"status {bad}, finite {bool(torch.isfinite(decoder.y).all())}")
    return bad


if __name__ == "__main__":
    sys.exit(main())
