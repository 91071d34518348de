"""A small hybrid model decoded in HBM: embedding lookup, layers of the gated
delta rule and of attention over a quantised paged cache with rotary positions,
the output head and the sampler, each through the framework's device calls.

    python examples/hybrid_decode.py --seqs 4 --prompt 40 --steps 16

The weights are random; the projections between the calls are plain torch
products. What it shows is how the pieces fit: one page table for the attention
layers, one state pool with a slot per sequence, prompts of different lengths and
single tokens through the same `step`.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-llm_amd"))
import rl_mixers  # noqa: E402
import rl_sampler  # noqa: E402

DEV = "cuda:0"


def q6k_tensor(g, rows, k):
    """A random Q6_K tensor: blocks of ql[128] qh[64] scales[16] d:f16."""
    blocks = rows * -(-k // 256)
    w = g.integers(0, 256, (blocks, 210), dtype=np.uint8)
    w[:, 192:208] = g.integers(-32, 32, (blocks, 16)).astype(np.int8).view(np.uint8)
    w[:, 208:] = np.frombuffer(np.float16(1.0 / 4096).tobytes(), np.uint8)
    return w.reshape(-1)


def norm(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


class HybridModel:
    """Layers "d" (delta rule) and "a" (attention), for up to `seqs` sequences of
    `context` tokens and calls of `max_rows` tokens."""

    def __init__(self, seqs, context, max_rows, layers="dda", hidden=512, vocab=4096, heads=8, kv_heads=2, dim=64,
                 key_heads=4, value_heads=8, page=16, cache="i8", seed=0):
        g = np.random.default_rng(seed)
        self.layers, self.hidden, self.vocab, self.page = layers, hidden, vocab, page
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        self.key_heads, self.value_heads = key_heads, value_heads
        self.head = rl_sampler.DeviceHead(q6k_tensor(g, vocab, hidden), hidden, vocab, max_batch=max(max_rows, seqs))
        self.sampler = rl_sampler.DeviceSampler(seqs, vocab)

        def weight(n, m):
            return torch.from_numpy((g.standard_normal((n, m)) * n ** -0.5).astype(np.float32)).to(DEV)
        self.weights = []
        for kind in layers:
            if kind == "a":
                inputs = (heads + 2 * kv_heads) * dim
                self.weights.append((weight(hidden, inputs), weight(heads * dim, hidden)))
            else:
                inputs = (2 * key_heads + value_heads) * dim + 2 * value_heads
                self.weights.append((weight(hidden, inputs), weight(value_heads * dim, hidden)))
        self.width = -(-context // page)
        self.rotary = rl_mixers.DeviceRotary(dim // 2, base=1e6)  # half of each head is turned
        self.caches = [rl_mixers.DeviceCache(seqs * self.width, page, kv_heads, dim, cache) if kind == "a" else None
                       for kind in layers]
        self.states = [torch.zeros(seqs, value_heads, dim, dim, device=DEV) if kind == "d" else None for kind in layers]
        self.attention = rl_mixers.DeviceAttention(max_rows, heads, kv_heads, dim, context)
        self.delta = rl_mixers.DeviceDelta(max_rows, seqs, key_heads, value_heads, dim, dim)
        # Every sequence has its pages from the start, in a shuffled order; a server would hand them out as it goes.
        order = torch.from_numpy(g.permutation(seqs * self.width).astype(np.int32)).to(DEV)
        self.table = order.view(seqs, self.width)
        self.lens = [0] * seqs

    def hidden_rows(self, tokens, counts):
        """tokens int32 [rows], counts[i] new ones of each sequence (0 or more);
        the rows before the output head."""
        seqs, rows = len(counts), int(sum(counts))
        starts = torch.tensor(np.cumsum([0] + list(counts)), dtype=torch.int32, device=DEV)
        places = np.concatenate([np.arange(n, n + c) for n, c in zip(self.lens, counts)])
        sequence = torch.from_numpy(np.repeat(np.arange(seqs), counts)).to(DEV)
        positions = torch.from_numpy(places).to(DEV)
        slots = self.table[sequence, positions // self.page].long() * self.page + positions % self.page
        self.lens = [n + c for n, c in zip(self.lens, counts)]
        lens = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        own = torch.arange(seqs, dtype=torch.int32, device=DEV)
        most = max(counts)
        x = 0.2 * norm(self.head.embed(tokens))
        for kind, (w_in, w_out), cache, states in zip(self.layers, self.weights, self.caches, self.states):
            y = norm(x) @ w_in
            if kind == "a":
                q, k, v = (t.view(rows, -1, self.dim) for t in y.split(
                    [self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim], 1))
                turned, out = torch.empty(q.shape, device=DEV), torch.empty(q.shape, device=DEV)
                self.rotary.apply(q, positions, turned)
                cache.write(k, v, slots, rotary=self.rotary, positions=positions)
                self.attention.rows(cache, turned, out, lens, self.table, starts=starts, most_rows=most)
            else:
                kd, vd = self.key_heads * self.dim, self.value_heads * self.dim
                q, k, v, gate, beta = y.split([kd, kd, vd, self.value_heads, self.value_heads], 1)
                q, k, v = (t.view(rows, -1, self.dim) for t in (q, k, v))
                out = torch.empty(v.shape, device=DEV)
                gate, beta = -torch.nn.functional.softplus(gate), torch.sigmoid(beta)
                self.delta.rows(q, k, v, gate, beta, out, states, own, own, starts, normalise=True, most_rows=most)
            x = x + out.view(rows, -1) @ w_out
        return norm(x)

    def step(self, tokens, counts, settings, uniforms):
        """One call of the model; the next token of every sequence, int32 [seqs]."""
        last = torch.tensor(np.cumsum(counts) - 1, device=DEV)
        logits = self.head.logits(self.hidden_rows(tokens, counts)[last].contiguous())
        n = len(counts)
        token = torch.empty(n, dtype=torch.int32, device=DEV)
        kept, used = torch.empty_like(token), torch.empty(n, dtype=torch.uint8, device=DEV)
        self.sampler.configure([settings] * n)
        self.sampler.sample_rows(logits, n, logits.stride(0), token, kept, used, uniforms=uniforms, vocab=self.vocab)
        return token


def decode(seqs=4, prompt=40, steps=16, seed=0, cache="i8"):
    """Prompts of up to `prompt` random tokens, then `steps` drawn ones each:
    [seqs][steps]."""
    g = np.random.default_rng(seed)
    counts = [int(n) for n in g.integers(1, prompt + 1, seqs)]
    model = HybridModel(seqs, prompt + steps, max(sum(counts), seqs), cache=cache, seed=seed)
    settings = rl_sampler.sampling(temperature=0.8, top_k=40, top_p=0.95)
    draws = torch.from_numpy(g.random((steps, seqs)).astype(np.float32)).to(DEV)
    tokens = torch.from_numpy(g.integers(0, model.vocab, sum(counts)).astype(np.int32)).to(DEV)
    out = []
    for i in range(steps):
        tokens = model.step(tokens, counts, settings, draws[i])
        counts = [1] * seqs
        out.append(tokens)
    return torch.stack(out, 1).cpu().numpy()


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=40)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--cache", default="i8", choices=["bf16", "f16", "i8", "f8"])
    a = ap.parse_args()
    for i, row in enumerate(decode(a.seqs, a.prompt, a.steps, a.seed, a.cache)):
        print("sequence %d: %s" % (i, " ".join(map(str, row))))
