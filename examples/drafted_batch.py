"""A batch that shares a prompt, decoded with drafted tokens: layers of the short
convolution and the state space scan and of attention behind the shared prompt, the
output head, the sampler, and the verification of what an early exit drafts.

    python examples/drafted_batch.py --seqs 4 --prompt 100 --steps 8 --drafts 3

The weights are random, hence the high temperature; the projections between the calls
are plain torch products.
What it shows is how the pieces fit: the prompt runs once and leaves its states in a
slot that every sequence begins from and its keys and values in pages that all read; a
step drafts with the first layer alone, runs all rows through the model without keeping
the states, verifies the sampler's candidates, and then advances the states by what was
accepted.
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rust-llm_amd"))
sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import rl_drafts  # noqa: E402
import rl_mixers  # noqa: E402
import rl_sampler  # noqa: E402
from hybrid_decode import norm, q6k_tensor  # noqa: E402

DEV = "cuda:0"


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device=DEV)


class DraftedModel:
    """`layers`: "s" for the convolution and the scan, "a" for attention; the first is
    the drafter's."""

    def __init__(self, seqs, prompt, own, drafts, layers="ssa", hidden=256, vocab=4096, channels=384, state=16, heads=8,
                 kv_heads=2, dim=64, page=16, cache="i8", keep=32, seed=0):
        g = np.random.default_rng(seed)
        gen = torch.Generator(device=DEV)
        gen.manual_seed(seed)

        def weight(*shape):
            return torch.randn(shape, generator=gen, device=DEV) * shape[-2] ** -0.5

        self.seqs, self.layers, self.vocab, self.keep, self.page = seqs, layers, vocab, keep, page
        self.channels, self.state, self.heads, self.kv_heads, self.dim = channels, state, heads, kv_heads, dim
        rows = max(prompt, seqs * (drafts + 1))
        self.head = rl_sampler.DeviceHead(q6k_tensor(g, vocab, hidden), hidden, vocab, max_batch=rows)
        self.rotary = rl_mixers.DeviceRotary(dim // 2, base=1e6)
        self.weights, self.mixers, self.pools = [], [], []
        pages, own_pages = -(-prompt // page), -(-own // page)
        order = np.random.default_rng(seed + 1).permutation(pages + seqs * own_pages).astype(np.int32)
        self.prefix_table, self.table = i32(order[:pages][None]), i32(order[pages:].reshape(seqs, own_pages))
        for kind in layers:
            if kind == "s":
                # x, z, a step a channel, b and c; from the convolution's output but z
                self.weights.append([weight(hidden, 2 * channels), weight(channels, channels + 2 * state), weight(channels, hidden)])
                a = -torch.arange(1, state + 1, dtype=torch.float32).expand(channels, state)
                conv = rl_mixers.DeviceConv(torch.from_numpy(g.uniform(-0.5, 0.5, (channels, 4)).astype(np.float32)))
                scan = rl_mixers.DeviceScan(rows, seqs, a, skip=torch.ones(channels),
                                            dt_bias=torch.from_numpy(g.uniform(-5, -2, channels).astype(np.float32)))
                self.mixers.append((conv, scan))
                # A slot a sequence, one each for the drafter, and the prompt's.
                self.pools.append((torch.zeros(2 * seqs + 1, 3, channels, device=DEV),
                                   torch.zeros(2 * seqs + 1, channels, state, device=DEV)))
            else:
                self.weights.append([weight(hidden, (heads + 2 * kv_heads) * dim), weight(heads * dim, hidden)])
                self.mixers.append((rl_mixers.DeviceCache(len(order), page, kv_heads, dim, cache),
                                    rl_mixers.DeviceAttention(rows, heads, kv_heads, dim, max(prompt, own))))
                self.pools.append(None)
        self.sampler = rl_sampler.DeviceSampler(rows, vocab)
        self.settings = rl_sampler.sampling(temperature=4.0, top_k=keep, top_p=0.95)
        self.verifier = rl_drafts.DeviceDrafts(seqs, vocab)
        self.own = torch.arange(seqs, dtype=torch.int32, device=DEV)
        self.none, self.scratch, self.prompt_slot = torch.full_like(self.own, -1), self.own + seqs, 2 * seqs
        self.prompt, self.lens = prompt, [0] * seqs

    def mix(self, i, y, into, to, starts, most):
        """The convolution and the scan of layer i over projected rows, from and to slots."""
        conv, scan = self.mixers[i]
        x, z = (t.contiguous() for t in y.split(self.channels, 1))
        u, out = torch.empty_like(x), torch.empty_like(x)
        conv.rows(x, u, self.pools[i][0], into, to, starts)
        dt, b, c = (u @ self.weights[i][1]).split([self.channels, self.state, self.state], 1)
        scan.rows(u, dt, b[:, None], c[:, None], out, self.pools[i][1], into, to, starts, z=z, most_rows=most)
        return out @ self.weights[i][2]

    def run(self, tokens, counts, into, to, layers=None, prompt=False):
        """The rows before the head of counts[s] tokens of each sequence (or of the
        prompt), and the projected rows of the "s" layers. Attention layers write the
        tokens' keys and values behind those of lens."""
        starts, rows, most = i32(np.cumsum([0] + list(counts))), int(sum(counts)), max(counts)
        first = [0] if prompt else self.lens
        places = np.concatenate([np.arange(n, n + c) for n, c in zip(first, counts)])
        at = torch.as_tensor(places, device=DEV)
        table = self.prefix_table if prompt else self.table
        sequence = torch.as_tensor(np.repeat(np.arange(len(counts)), counts), device=DEV)
        slots = table[sequence, at // self.page].long() * self.page + at % self.page
        positions = at if prompt else at + self.prompt
        lens = i32([n + c for n, c in zip(first, counts)])
        x, saved = 0.2 * norm(self.head.embed(tokens)), []
        for i, kind in enumerate(self.layers[:layers]):
            y = norm(x) @ self.weights[i][0]
            if kind == "s":
                saved.append(y)
                x = x + self.mix(i, y, into, to, starts, most)
                continue
            cache, attention = self.mixers[i]
            q, k, v = (t.view(rows, -1, self.dim) for t in y.split(
                [self.heads * self.dim, self.kv_heads * self.dim, self.kv_heads * self.dim], 1))
            turned, out = torch.empty(q.shape, device=DEV), torch.empty(q.shape, device=DEV)
            self.rotary.apply(q, positions, turned)
            cache.write(k, v, slots, rotary=self.rotary, positions=positions)
            if prompt:
                attention.rows(cache, turned, out, lens, table, starts=starts, most_rows=most)
            else:
                attention.shared(cache, turned, out, lens, table, i32([0, self.seqs]), i32([self.prompt]), self.prefix_table,
                                 starts=starts, most_rows=most)
            x = x + out.view(rows, -1) @ self.weights[i][1]
        return norm(x), saved

    def read_prompt(self, tokens):
        """Runs the prompt once; every sequence begins from its states."""
        slot = i32([self.prompt_slot])
        hidden, _ = self.run(tokens, [len(tokens)], slot - slot - 1, slot, prompt=True)
        for pools in self.pools:
            for pool in pools or ():
                pool[:self.seqs] = pool[self.prompt_slot]
        return hidden

    def draw(self, hidden, uniforms):
        """A token a row, and the candidates that it was drawn from."""
        rows = hidden.shape[0]
        logits = self.head.logits(hidden)
        token, kept = (torch.empty(rows, dtype=torch.int32, device=DEV) for _ in range(2))
        used = torch.empty(rows, dtype=torch.uint8, device=DEV)
        ids, probs = torch.empty(rows, self.keep, dtype=torch.int32, device=DEV), torch.empty(rows, self.keep, device=DEV)
        self.sampler.configure([self.settings] * rows)
        self.sampler.sample_rows(logits, rows, logits.stride(0), token, kept, used, uniforms=uniforms, out_ids=ids,
                                 out_probs=probs, cand_stride=self.keep)
        return token, ids, probs, kept

    def step(self, last, drafts, g):
        """From each sequence's last token, `drafts` drafted ones: the tokens of each,
        [seqs][drafts + 1] with -1 after the last, and the accepted drafts."""
        n = self.seqs

        def uniform(rows):
            return torch.from_numpy(g.random(rows).astype(np.float32)).to(DEV)

        token, said = last, []
        for j in range(drafts):  # one layer, its states in slots of its own
            hidden, _ = self.run(token, [1] * n, self.own if j == 0 else self.scratch, self.scratch, layers=1)
            said.append(self.draw(hidden, uniform(n)))
            token = said[-1][0]
        drafted, ids, probs, kept = (torch.stack(t, 1).flatten(0, 1) for t in zip(*said))
        rows = torch.cat([last[:, None], drafted.view(n, drafts)], 1).flatten()
        hidden, saved = self.run(rows, [drafts + 1] * n, self.own, self.none)
        _, target_ids, target, target_kept = self.draw(hidden, uniform(rows.shape[0]))
        accepted, tokens = torch.empty_like(self.own), torch.empty_like(rows)
        self.verifier.verify(target, drafted, i32(np.arange(n + 1) * drafts), uniform(n * drafts), uniform(n), accepted,
                             tokens, draft=probs, target_ids=target_ids, target_kept=target_kept, draft_ids=ids,
                             draft_kept=kept)
        # The states go on by the tokens that stand: the last one and the accepted drafts.
        counts = (accepted + 1).tolist()
        stands = torch.as_tensor(np.concatenate([s * (drafts + 1) + np.arange(c) for s, c in enumerate(counts)]), device=DEV)
        for i, y in zip([i for i, kind in enumerate(self.layers) if kind == "s"], saved):
            self.mix(i, y[stands], self.own, self.own, i32(np.cumsum([0] + counts)), max(counts))
        self.lens = [a + c for a, c in zip(self.lens, counts)]
        return tokens.view(n, drafts + 1), accepted


def decode(seqs=4, prompt=100, steps=8, drafts=3, seed=0, cache="i8"):
    """The tokens of each sequence after a random prompt, and the accepted drafts."""
    g = np.random.default_rng(seed)
    model = DraftedModel(seqs, prompt, steps * (drafts + 1), drafts, cache=cache, seed=seed)
    hidden = model.read_prompt(torch.from_numpy(g.integers(0, model.vocab, prompt).astype(np.int32)).to(DEV))
    first, _, _, _ = model.draw(hidden[-1:].expand(seqs, -1).contiguous(), torch.from_numpy(g.random(seqs).astype(np.float32)).to(DEV))
    last, said, accepted = first, [[int(t)] for t in first], 0
    for _ in range(steps):
        tokens, count = model.step(last, drafts, g)
        last = tokens.gather(1, count[:, None].long())[:, 0].contiguous()
        accepted += int(count.sum())
        for s, (row, c) in enumerate(zip(tokens.tolist(), count.tolist())):
            said[s] += row[:c + 1]
    return said, accepted


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=100)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--drafts", type=int, default=3)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--cache", default="i8", choices=["bf16", "i8", "f8"])
    a = ap.parse_args()
    said, accepted = decode(a.seqs, a.prompt, a.steps, a.drafts, a.seed, a.cache)
    for i, row in enumerate(said):
        print("sequence %d: %s" % (i, " ".join(map(str, row))))
    print("%d of %d drafts accepted" % (accepted, a.seqs * a.steps * a.drafts))
