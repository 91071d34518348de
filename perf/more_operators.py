"""What is timed of the operators that a serving step of a hybrid model runs beside
those of operators.py: its batch shares a prompt, its layers scan, and it drafts.

  conv     the short causal convolution in front of the delta rule or of a scan
  scan     the selective state space scan: one step of a batch, a verify, prompts
  shared   attention of a batch whose sequences share long prefixes of the cache
  drafts   verification of drafted tokens against the target's probabilities

The plain forms are elementary torch operations in f32 (f64 for the sums that a
drawn token depends on), rounded once to the output's type. Sequence lengths follow
from the case alone; their order, the pages' order and all values follow from the
seed. States are read from one half of a pool and written to the other, as a
program does that may have to go back to the state before a verify, so a pass can
be repeated.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
WIDTH = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "f8": 1}


def _conv(name, seqs, shortest, longest, channels, width, dtype, act="silu"):
    return {"name": name, "op": "conv", "seqs": seqs, "shortest": shortest, "longest": longest, "channels": channels,
            "width": width, "dtype": dtype, "act": act}


def _scan(name, seqs, shortest, longest, channels, groups, state, dtype, gated=True):
    return {"name": name, "op": "scan", "seqs": seqs, "shortest": shortest, "longest": longest, "channels": channels,
            "groups": groups, "state": state, "dtype": dtype, "gated": gated}


def _shared(name, groups, prefix, seqs, shortest, longest, rows, q_heads, kv_heads, dim, page, fmt, dtype):
    return {"name": name, "op": "shared", "groups": groups, "prefix": prefix, "seqs": seqs, "shortest": shortest,
            "longest": longest, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "format": fmt, "dtype": dtype}


def _drafts(name, seqs, shortest, longest, vocab, form, keep=0):
    return {"name": name, "op": "drafts", "seqs": seqs, "shortest": shortest, "longest": longest, "vocab": vocab,
            "form": form, "keep": keep}


def listed():
    return [
        # One token of one sequence: all launch and latency.
        _conv("conv_1", 1, 1, 1, 8192, 4, "bf16"),
        # A long prompt, the queries, keys and values of 16 / 32 heads of 128.
        _conv("conv_prompt_8192", 1, 8192, 8192, 8192, 4, "bf16"),
        # A few prompts of odd lengths in f32, an odd number of channels.
        _conv("conv_ragged_7", 7, 33, 701, 2027, 3, "f32", act="none"),
        # The step of a serving batch: states in and out, one token each.
        _scan("scan_64", 64, 1, 1, 5120, 1, 16, "bf16"),
        # A long prompt of one sequence: its length has to be shared out.
        _scan("scan_prompt_8192", 1, 8192, 8192, 5120, 1, 16, "bf16"),
        # A few prompts of odd lengths in f32, groups of channels, larger states.
        _scan("scan_ragged_24", 24, 33, 701, 1536, 4, 32, "f32", gated=False),
        # A small batch over a system prompt: the smallest call.
        _shared("shared_8", 1, 1009, 8, 16, 128, 1, 16, 4, 256, 32, "bf16", "bf16"),
        # The step of a serving batch over one long document.
        _shared("shared_64", 1, 16384, 64, 16, 512, 1, 32, 8, 128, 64, "bf16", "bf16"),
        # The check of four drafted tokens over three prompts in an int8 cache,
        # pages of 24 tokens (they end inside any tile).
        _shared("shared_verify_96", 3, 8001, 96, 16, 512, 5, 32, 8, 128, 24, "i8", "bf16"),
        # Eight drafted tokens of one sequence, whole rows of probabilities.
        _drafts("drafts_1", 1, 8, 8, 151936, "dense"),
        # A serving batch with up to four drafted tokens each, a large vocabulary.
        _drafts("drafts_64", 64, 1, 4, 248320, "dense"),
        # The same over the candidates that a sampler keeps.
        _drafts("drafts_lists_64", 64, 2, 8, 151936, "lists", keep=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_lengths(rng, kind, seqs, rows):
    longest = {"step": 1, "verify": rng.choice([2, 5, 9, 17]), "prompt": _log_int(rng, 32, max(32, rows // seqs))}[kind]
    return (max(1, longest // rng.choice([1, 2, 16])) if kind == "prompt" else longest), longest


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "shared", "shared", "drafts"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    kind = rng.choice(["step", "verify", "prompt", "prompt"])
    seqs = _log_int(rng, 1, 96) if kind != "prompt" else _log_int(rng, 1, 24)
    if op == "conv":
        shortest, longest = _draw_lengths(rng, kind, seqs, 8192)
        c = _conv("", seqs, shortest, longest, rng.choice([1, 2, 8, 8, 8]) * _log_int(rng, 64, 512) + rng.choice([0, 0, 1]),
                  rng.choice([2, 3, 4, 4, 4]), dtype, rng.choice(["silu", "silu", "none"]))
    elif op == "scan":
        groups, state = rng.choice([1, 1, 2, 4]), rng.choice([16, 16, 16, 8, 32, 64])
        # At most the longest listed case's products of channels, state values and tokens.
        channels = groups * max(8, _log_int(rng, 128, 81920 // state) // groups)
        rows = min(8192, 8192 * 5120 * 16 // (channels * state))
        shortest, longest = _draw_lengths(rng, kind, seqs, rows)
        c = _scan("", seqs, shortest, longest, channels, groups, state, dtype, rng.random() < 0.7)
    elif op == "shared":
        seqs, kv_heads, rows = _log_int(rng, 2, 128), rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 1, 2, 5, 9])
        dim, groups = rng.choice([64, 80, 96, 128, 256]), min(seqs, rng.choice([1, 1, 2, 3, 8]))
        heads = kv_heads * rng.choice([1, 2, 4, 8] if rows <= 2 else [1, 2, 4])
        # At most the largest listed case's products of prefix, rows and heads.
        most = max(64, min(32768, 8001 * 96 * 5 * 32 * 128 // (seqs * rows * heads * dim)))
        fmt = rng.choice(["i8", "f8", "same", "same", "same"])
        longest = _log_int(rng, 16, min(1024, (1 << 24) // (seqs * kv_heads * dim)))
        c = _shared("", groups, _log_int(rng, 64, most), seqs, max(1, rows, longest // rng.choice([1, 4, 32])),
                    max(rows, longest), rows, heads, kv_heads, dim, rng.choice([16, 24, 32, 64, 128]),
                    ("f16" if dtype == "f16" else "bf16") if fmt == "same" else fmt, dtype)
    else:
        longest = rng.choice([1, 2, 4, 8, 16])
        shortest, form = rng.choice([longest, max(0, longest // 2), 0]), rng.choice(["dense", "dense", "lists", "greedy"])
        # At most the largest listed case's rows.
        vocab = rng.choice([151936, 248320, _log_int(rng, 1000, 248320)])
        seqs = _log_int(rng, 1, max(1, min(128, 64 * 4 * 248320 // (vocab * longest))))
        c = _drafts("", seqs, shortest, longest, vocab, form, _log_int(rng, 2, 400) if form == "lists" else 0)
    del c["name"]
    return c


def _spread(case):
    # Lengths from the shortest to the longest: evenly, or where they are long over their logarithm.
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    if n == 1:
        return [b]
    if case["op"] == "drafts":
        return [a + (b - a) * i // (n - 1) for i in range(n)]
    return [int(round(a * (b / a) ** (i / (n - 1)))) for i in range(n)]


def _prefixes(case):
    """(tokens of each group's prefix, the groups' first sequences and the end)."""
    n = case["groups"]
    return [max(1, case["prefix"] // (i + 1)) for i in range(n)], [case["seqs"] * i // n for i in range(n + 1)]


def work(case):
    op = case["op"]
    if op == "drafts":
        # One row of each side a sequence, where the drawn token comes from.
        values = case["seqs"] * (case["keep"] or case["vocab"])
        sides = 1 if case["form"] == "greedy" else 2
        return {"bytes": sides * values * (8 if case["form"] == "lists" else 4), "flops": 3 * values}
    rows, size = sum(_spread(case)), WIDTH[case["dtype"]]
    if op == "conv":
        return {"bytes": (2 * rows + 2 * case["seqs"] * (case["width"] - 1)) * case["channels"] * size,
                "flops": 2 * rows * case["channels"] * case["width"]}
    if op == "scan":
        values = rows * case["channels"]
        return {"bytes": (values * (4 if case["gated"] else 3) + 2 * rows * case["groups"] * case["state"]) * size
                + 8 * case["seqs"] * case["channels"] * case["state"],
                "flops": 6 * values * case["state"]}
    lens, (prefix, first) = _spread(case), _prefixes(case)
    code = case["dim"] * WIDTH[case["format"]] + (4 if WIDTH[case["format"]] == 1 else 0)
    heads = case["rows"] * case["q_heads"]
    seen = sum(lens) + sum(p * (b - a) for p, a, b in zip(prefix, first, first[1:]))
    return {"bytes": (sum(lens) + sum(prefix)) * case["kv_heads"] * 2 * code + 2 * case["seqs"] * heads * case["dim"] * size,
            "flops": 4 * seen * heads * case["dim"]}


# ---------------------------------------------------------------- inputs --
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * sigma).to(TYPES[dtype])


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device=DEV)


def _ordered(case, g):
    """The lengths in the seed's order, and where each sequence's rows start."""
    lens = torch.tensor(_spread(case), device=DEV)[torch.randperm(case["seqs"], generator=g, device=DEV)]
    return lens, torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(lens, 0)]).to(torch.int32)


def _inputs(case, seed):
    """The tensors that both forms start from."""
    g, op, n = _generator(seed), case["op"], case["seqs"]
    if op == "conv":
        lens, starts = _ordered(case, g)
        c = case["channels"]
        return {"lens": lens, "starts": starts, "x": _normal(g, (sum(_spread(case)), c), case["dtype"]),
                "weight": _rand(g, c, case["width"]) - 0.5, "bias": 0.2 * (_rand(g, c) - 0.5),
                "states": _normal(g, (2 * n, case["width"] - 1, c), case["dtype"])}
    if op == "scan":
        lens, starts = _ordered(case, g)
        rows, c, m, dtype = sum(_spread(case)), case["channels"], case["state"], case["dtype"]
        s = {"lens": lens, "starts": starts,
             # Decays of 1 to m a unit of step, steps from 0.001 to 0.1 by channel.
             "a": -torch.arange(1, m + 1, device=DEV) * (0.1 * torch.randn((c, m), generator=g, device=DEV)).exp(),
             "skip": 1 + 0.1 * torch.randn((c,), generator=g, device=DEV)}
        step = (math.log(0.001) + _rand(g, c) * math.log(100.0)).exp()
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["x"], s["dt"] = _normal(g, (rows, c), dtype), _normal(g, (rows, c), dtype, 0.5)
        s["b"], s["c"] = (_normal(g, (rows, case["groups"], m), dtype) for _ in range(2))
        s["z"] = _normal(g, (rows, c), dtype) if case["gated"] else None
        s["states"] = 0.3 * torch.randn((2 * n, c, m), generator=g, device=DEV)
        return s
    if op == "shared":
        lens, (prefix, first) = torch.tensor(_spread(case), device=DEV), _prefixes(case)
        lens = lens[torch.randperm(n, generator=g, device=DEV)]
        page = case["page"]
        need = [-(-p // page) for p in prefix]
        own_need = -(-lens // page)
        pages = sum(need) + sum(-(-t // page) for t in _spread(case))
        order = torch.randperm(pages, generator=g, device=DEV)

        def table(count, begin, widest):  # [rows][widest]: `count` pages of the shuffled ones from `begin` on
            j = torch.arange(widest, device=DEV)
            at = (begin[:, None] + j).clamp(max=pages - 1)
            return torch.where(j < count[:, None], order[at], torch.zeros_like(at)).to(torch.int32)

        shared_need = torch.tensor(need, device=DEV)
        source = "f16" if case["format"] == "f16" else "bf16"
        shape = (pages * page, case["kv_heads"], case["dim"])
        return {"k": _normal(g, shape, source), "v": _normal(g, shape, source),
                "q": _normal(g, (n * case["rows"], case["q_heads"], case["dim"]), case["dtype"], 2.0),
                "lens": lens.to(torch.int32), "pages": pages,
                "prefix_table": table(shared_need, torch.cumsum(shared_need, 0) - shared_need, max(need)),
                "table": table(own_need, sum(need) + torch.cumsum(own_need, 0) - own_need, -(-case["longest"] // page)),
                "prefix_lens": torch.tensor(prefix, dtype=torch.int32, device=DEV),
                "groups": torch.tensor(first, dtype=torch.int32, device=DEV)}
    lens, starts = _ordered(case, g)
    drafts, vocab = sum(_spread(case)), case["vocab"]
    # Each draft's target row; a sequence has one row more than drafts.
    sequence = torch.repeat_interleave(torch.arange(n, device=DEV), lens)
    row = torch.arange(drafts, device=DEV) + sequence
    target = torch.randn((drafts + n, vocab), generator=g, device=DEV) * 3.0
    draft = (target[row] + 0.7 * torch.randn((drafts, vocab), generator=g, device=DEV)) if case["form"] != "greedy" else target[row]
    s = {"lens": lens, "starts": starts, "uniforms": _rand(g, drafts), "draws": _rand(g, n), "target_ids": None,
         "target_kept": None, "draft": None, "draft_ids": None, "draft_kept": None}
    for name, logits in (("target", target), ("draft", draft)):
        if case["form"] == "lists":
            most = min(case["keep"], vocab)
            top, ids = torch.topk(logits, most, dim=1)
            kept = torch.randint(max(1, most // 4), most + 1, (logits.shape[0],), generator=g, device=DEV)
            top = top.masked_fill(torch.arange(most, device=DEV) >= kept[:, None], -math.inf)
            s[name], s[name + "_ids"] = torch.softmax(top, 1), ids.to(torch.int32)
            s[name + "_kept"] = kept.to(torch.int32)
        elif name == "target" or case["form"] == "dense":
            s[name] = torch.softmax(logits, 1)
    if case["form"] == "greedy":  # a drafter without probabilities, right about half the time
        second = torch.topk(draft, 2, dim=1).indices
        pick = torch.randint(0, 2, (drafts,), generator=g, device=DEV)
        s["drafted"] = second.gather(1, pick[:, None])[:, 0].to(torch.int32)
    else:  # drawn from the draft's probabilities
        race = s["draft"] / torch.empty_like(s["draft"]).exponential_(generator=g)
        at = race.argmax(1)
        s["drafted"] = at.to(torch.int32) if case["form"] == "dense" else s["draft_ids"].gather(1, at[:, None])[:, 0]
    return s


def _encode(x, fmt):
    """f32 vectors as the cache holds them: (codes, a scale a vector or None)."""
    if fmt in TYPES:
        return x.to(TYPES[fmt]), None
    most = x.abs().amax(-1, keepdim=True)
    scale = most / torch.full_like(most, 127.0 if fmt == "i8" else 448.0)  # a quotient, no product with a reciprocal
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    if fmt == "i8":
        return torch.round(y).clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], op = case, case["op"]
    if own:
        return _prepare_own(s, case)
    if op == "shared":
        s["pool_k"], s["pool_v"] = _encode(s["k"].float(), case["format"]), _encode(s["v"].float(), case["format"])
        del s["k"], s["v"]
    return s


def _prepare_own(s, case):
    sys.path.insert(0, os.path.abspath("rust-llm_amd"))
    import rl_drafts
    import rl_mixers
    op, n = case["op"], case["seqs"]
    if op in ("conv", "scan"):
        slots = torch.arange(2 * n, dtype=torch.int32, device=DEV)
        s["before"], s["after"], s["states_after"] = slots[:n], slots[n:], s["states"][n:]
        s["out"] = torch.empty_like(s["x"])
    if op == "conv":
        s["conv"] = rl_mixers.DeviceConv(s["weight"], s["bias"], case["act"])
    elif op == "scan":
        s["scan"] = rl_mixers.DeviceScan(s["x"].shape[0], n, s["a"], groups=case["groups"], skip=s["skip"],
                                         dt_bias=s["dt_bias"])
    elif op == "shared":
        s["cache"] = rl_mixers.DeviceCache(s["pages"], case["page"], case["kv_heads"], case["dim"], case["format"])
        s["cache"].write(s["k"], s["v"], torch.arange(s["k"].shape[0], device=DEV))
        del s["k"], s["v"]
        s["attention"] = rl_mixers.DeviceAttention(s["q"].shape[0], case["q_heads"], case["kv_heads"], case["dim"],
                                                   max(case["longest"], case["prefix"]))
        s["starts"] = torch.arange(n + 1, dtype=torch.int32, device=DEV) * case["rows"]
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
    else:
        s["verify"] = rl_drafts.DeviceDrafts(n, case["vocab"])
        s["accepted"] = torch.empty(n, dtype=torch.int32, device=DEV)
        s["tokens"] = torch.empty(s["target"].shape[0], dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------- the passes --
def run(s):
    op = s["case"]["op"]
    if own:
        return {"conv": _own_conv, "scan": _own_scan, "shared": _own_shared, "drafts": _own_drafts}[op](s)
    return {"conv": _plain_conv, "scan": _plain_scan, "shared": _plain_shared, "drafts": _plain_drafts}[op](s)


def _own_conv(s):
    s["conv"].rows(s["x"], s["out"], s["states"], s["before"], s["after"], starts=s["starts"])
    return s["out"], s["states_after"]


def _own_scan(s):
    s["scan"].rows(s["x"], s["dt"], s["b"], s["c"], s["out"], s["states"], s["before"], s["after"], starts=s["starts"],
                   z=s["z"], most_rows=s["case"]["longest"])
    return s["out"], s["states_after"]


def _own_shared(s):
    c = s["case"]
    s["attention"].shared(s["cache"], s["q"], s["out"], s["lens"], s["table"], s["groups"], s["prefix_lens"],
                          s["prefix_table"], starts=s["starts"], lse=s["lse"], most_rows=c["rows"],
                          max_len=c["longest"], max_prefix=c["prefix"])
    return s["out"], s["lse"]


def _own_drafts(s):
    s["verify"].verify(s["target"], s["drafted"], s["starts"], s["uniforms"], s["draws"], s["accepted"], s["tokens"],
                       draft=s["draft"], target_ids=s["target_ids"], target_kept=s["target_kept"],
                       draft_ids=s["draft_ids"], draft_kept=s["draft_kept"])
    return s["accepted"], s["tokens"]


def _padded(s, longest):
    """(whether token t of sequence i is there, the row it has), [seqs][longest]."""
    t = torch.arange(longest, device=DEV)
    return t < s["lens"][:, None], (s["starts"][:-1].long()[:, None] + t).clamp(max=max(int(s["x"].shape[0]) - 1, 0))


def _plain_conv(s):
    c, n, w = s["case"], s["case"]["seqs"], s["case"]["width"]
    here, at = _padded(s, c["longest"])
    x = torch.cat([s["states"][:n].float(), s["x"].float()[at]], 1)  # [seqs][width - 1 + longest][channels]
    y = s["bias"].expand(n, c["longest"], -1)
    for j in range(w):
        y = y + s["weight"][:, j] * x[:, j:j + c["longest"]]
    if c["act"] == "silu":
        y = y / (1 + (-y).exp())
    last = s["lens"][:, None] + torch.arange(w - 1, device=DEV)
    states = x.gather(1, last[..., None].expand(-1, -1, x.shape[2]))
    return y[here].to(s["x"].dtype), states.to(s["x"].dtype)


def _plain_scan(s):
    """Pieces of about the square root of the length, all pieces of all sequences
    side by side: first each from a state of zeros, then with the state that the
    pieces before it leave."""
    c, n, m = s["case"], s["case"]["seqs"], s["case"]["state"]
    size = min(c["longest"], max(16, int(math.ceil(math.sqrt(c["longest"])))))
    pieces = -(-c["longest"] // size)
    here, at = _padded(s, pieces * size)
    per = c["channels"] // c["groups"]

    def cut(x):  # [size][seqs * pieces][...], zero past a sequence's end
        x = x.float()[at] * here.view(n, -1, *[1] * (x.dim() - 1))
        return x.view(n * pieces, size, *x.shape[2:]).movedim(1, 0)

    dt = s["dt"].float() + s["dt_bias"]
    dt = dt.clamp(min=0) + torch.log1p((-dt.abs()).exp())
    x, dt, b, cc = cut(s["x"]), cut(dt), cut(s["b"]), cut(s["c"])

    def spread(y):  # [...][groups][state] -> [...][channels][state]
        return y[:, :, None, :].expand(-1, -1, per, -1).reshape(y.shape[0], -1, m)

    def step(h, t):
        return h * (dt[t][..., None] * s["a"]).exp() + (dt[t] * x[t])[..., None] * spread(b[t])

    start = s["states"][:n]
    if pieces > 1:
        h = torch.zeros((n * pieces, c["channels"], m), device=DEV)
        for t in range(size):
            h = step(h, t)
        total = (dt.sum(0)[..., None] * s["a"]).exp().view(n, pieces, -1, m)
        h, starts = h.view(n, pieces, -1, m), []
        for j in range(pieces):
            starts.append(start)
            start = start * total[:, j] + h[:, j]
        h = torch.stack(starts, 1).flatten(0, 1)
    else:
        h = start
    out = torch.empty_like(x)
    for t in range(size):
        h = step(h, t)
        out[t] = (h * spread(cc[t])).sum(-1)
    out = out + s["skip"] * x
    if pieces == 1:
        start = h
    out = out.movedim(0, 1).reshape(n, pieces * size, -1)[here]
    if c["gated"]:
        z = s["z"].float()
        out = out * (z / (1 + (-z).exp()))
    return out.to(s["x"].dtype), start


def _plain_shared(s):
    c = s["case"]
    n, r, kv, page, dim = c["seqs"], c["rows"], c["kv_heads"], c["page"], c["dim"]
    group = c["q_heads"] // kv
    prefix, first = _prefixes(c)

    def gathered(pool, table, tokens):  # [...][kv heads][tokens][dim]
        t = torch.arange(tokens, device=DEV)
        slots = table.long()[..., t // page] * page + t % page
        codes, scale = pool
        x = (codes.view(torch.int8)[slots].view(codes.dtype) if codes.element_size() == 1 else codes[slots]).float()
        return (x if scale is None else x * scale[slots]).transpose(-3, -2).contiguous()

    def joined(q, pool, table, tokens, seen):  # maximum, sum and sum of values of the last axes but one
        x = torch.matmul(q, gathered(s[pool + "k"], table, tokens).transpose(-2, -1).contiguous()) * dim ** -0.5
        x = x if seen is None else x.masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = (x - top.clamp(min=-3e38)).exp()
        return top, p.sum(-1, keepdim=True), torch.matmul(p, gathered(s[pool + "v"], table, tokens))

    q = s["q"].float().view(n, r, kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n, kv, r * group, dim)
    at = s["lens"].long()[:, None] - r + torch.arange(r, device=DEV)  # [seqs][rows]
    seen = (torch.arange(c["longest"], device=DEV) <= at[..., None])[:, None, :, None, :]
    own_part = joined(q, "pool_", s["table"], c["longest"], seen.expand(n, 1, r, group, -1).reshape(n, 1, r * group, -1))
    parts = []
    for i, tokens in enumerate(prefix):
        a, b = first[i], first[i + 1]
        part = joined(q[a:b].transpose(0, 1).reshape(kv, -1, dim), "pool_", s["prefix_table"][i], tokens, None)
        parts.append([y.view(kv, b - a, r * group, -1).transpose(0, 1) for y in part])
    shared = [torch.cat(y) for y in zip(*parts)]
    top = torch.maximum(own_part[0], shared[0])
    f, g = (own_part[0] - top).exp(), (shared[0] - top).exp()
    total = own_part[1] * f + shared[1] * g
    o = (own_part[2] * f + shared[2] * g) / total

    def rows_first(y):
        return y.view(n, kv, r, group, -1).permute(0, 2, 1, 3, 4).reshape(n * r, c["q_heads"], -1)
    return rows_first(o).to(s["q"].dtype), rows_first(top + total.log())[..., 0].contiguous()


def _plain_drafts(s):
    """In f64: a drawn token depends on the last bits of long sums."""
    n, most = s["case"]["seqs"], s["case"]["longest"]
    lens, starts, lists = s["lens"], s["starts"].long(), s["target_ids"] is not None
    drafts = s["drafted"].shape[0]
    tokens = torch.full((drafts + n,), -1, dtype=torch.int32, device=DEV)
    i = torch.arange(max(most, 1), device=DEV)
    here = i < lens[:, None]
    at = (starts[:-1, None] + i).clamp(max=max(drafts - 1, 0))  # [seqs][most]
    if drafts:
        d = s["drafted"][at].long()
        row = torch.where(here, at + torch.arange(n, device=DEV)[:, None], 0)
        if lists:
            def of(name, where):
                found = s[name + "_ids"][where] == d[..., None]
                found &= torch.arange(found.shape[2], device=DEV) < s[name + "_kept"][where][..., None]
                return (s[name][where].double() * found).sum(-1)
            p, q = of("target", row), of("draft", at)
        else:
            p = s["target"][row, d].double()
            q = s["draft"][at, d].double() if s["draft"] is not None else torch.ones_like(p)
        fine = (s["uniforms"][at].double() * q < p) & here
        accepted = fine.long().cumprod(1).sum(1)
    else:
        accepted = torch.zeros(n, dtype=torch.int64, device=DEV)
    rejected = accepted < lens
    row = starts[:-1] + torch.arange(n, device=DEV) + accepted
    last = (starts[:-1] + accepted).clamp(max=max(drafts - 1, 0))  # the draft that was rejected
    p = s["target"][row].double()
    if lists:
        p = p * (torch.arange(p.shape[1], device=DEV) < s["target_kept"][row][:, None])
        q = s["draft"][last].double() * (torch.arange(s["draft"].shape[1], device=DEV) < s["draft_kept"][last][:, None])
        same = s["target_ids"][row][:, :, None] == s["draft_ids"][last][:, None, :]
        q = (same * q[:, None, :]).sum(-1)
    elif s["draft"] is not None:
        q = s["draft"][last].double() if drafts else torch.zeros_like(p)
    else:
        q = torch.zeros_like(p)
        if drafts:
            q.scatter_(1, s["drafted"][last].long()[:, None], 1.0)
    left = (p - q * rejected[:, None]).clamp(min=0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
    total = left.cumsum(1)
    drawn = (total > s["draws"].double()[:, None] * total[:, -1:]).long().argmax(1)
    if lists:
        drawn = s["target_ids"][row, drawn].long()
    if drafts:
        keep = i < accepted[:, None]
        tokens[(at + torch.arange(n, device=DEV)[:, None])[keep]] = s["drafted"][at[keep]]
    tokens[row] = drawn.to(torch.int32)
    return accepted.to(torch.int32), tokens


# ------------------------------------------------------ the same in 64 bits --
def exact(case, seed):
    s = _inputs(case, seed)
    return {"conv": _exact_conv, "scan": _exact_scan, "shared": _exact_shared, "drafts": _exact_drafts}[case["op"]](case, s)


def _exact_conv(case, s):
    w, out, states = case["width"], [], []
    kernel = s["weight"].double().t()  # [width][channels]
    for i, n in enumerate(s["lens"].tolist()):
        a = int(s["starts"][i])
        x = torch.vstack([s["states"][i].double(), s["x"][a:a + n].double()])
        y = (x.unfold(0, w, 1) * kernel.t()).sum(-1) + s["bias"].double()
        out.append(y * torch.sigmoid(y) if case["act"] == "silu" else y)
        states.append(x[n:])
    return torch.cat(out), torch.stack(states)


def _exact_scan(case, s):
    n, per = case["seqs"], case["channels"] // case["groups"]
    step = torch.nn.functional.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=40.0)
    drive = step * s["x"].double()
    a, b, c = s["a"].double(), s["b"], s["c"]
    starts, lens = s["starts"][:-1].tolist(), s["lens"].tolist()
    order = sorted(range(n), key=lambda i: -lens[i])  # the longest first: those still running lead
    h, first = s["states"][:n].double()[order], torch.tensor([starts[i] for i in order], device=DEV)
    out = s["skip"].double() * s["x"].double()
    for t in range(max(lens)):
        m = sum(1 for i in lens if i > t)
        at = first[:m] + t
        now = torch.exp(step[at].unsqueeze(-1) * a) * h[:m]
        now += drive[at].unsqueeze(-1) * b[at].double().repeat_interleave(per, 1)
        h[:m] = now
        out[at] += torch.einsum("ign,igpn->igp", c[at].double(), now.unflatten(1, (-1, per))).flatten(1)
    if case["gated"]:
        out *= torch.nn.functional.silu(s["z"].double())
    back = torch.empty_like(h)
    back[order] = h
    return out, back


def _exact_shared(case, s):
    r, page, kv = case["rows"], case["page"], case["kv_heads"]

    def stored(x):
        if case["format"] in TYPES:
            return x.to(TYPES[case["format"]]).double()
        # The step and the quotient that is rounded to a code are f32 by definition: halves occur.
        step = (x.double().abs().amax(-1, keepdim=True) / (127 if case["format"] == "i8" else 448)).float().double()
        y = (x.double() / torch.where(step > 0, step, 1.0)).float()
        return step * (y.double().round() if case["format"] == "i8" else y.to(torch.float8_e4m3fn).double())

    def slots(pages, n):
        t = torch.arange(n, device=DEV)
        return pages.long()[t // page] * page + t % page

    out, lse, group_of = [], [], torch.bucketize(torch.arange(case["seqs"], device=DEV), s["groups"][1:], right=True).tolist()
    held, last = None, -1
    prefix = s["prefix_lens"].tolist()
    for i, n in enumerate(s["lens"].tolist()):
        j = group_of[i]
        if j != last:
            at = slots(s["prefix_table"][j], prefix[j])
            held, last = [stored(s[x][at]).movedim(1, 0) for x in ("k", "v")], j  # [kv][tokens][dim]
        at = slots(s["table"][i], n)
        k, v = (torch.cat([old, stored(s[x][at]).movedim(1, 0)], 1) for x, old in zip(("k", "v"), held))
        q = s["q"][i * r:(i + 1) * r].double().view(r, kv, -1, case["dim"]).movedim(1, 0).flatten(1, 2)
        x = q @ k.transpose(1, 2) / math.sqrt(case["dim"])
        stands = (n - r + torch.arange(r, device=DEV)).repeat_interleave(case["q_heads"] // kv)[:, None]
        x[:, torch.arange(-prefix[j], n, device=DEV) > stands.clamp(min=-1)] = -math.inf
        out.append((torch.softmax(x, -1) @ v).unflatten(1, (r, -1)).movedim(0, 1).flatten(1, 2))
        lse.append(torch.logsumexp(x, -1).unflatten(1, (r, -1)).movedim(0, 1).flatten(1, 2))
    return torch.cat(out), torch.cat(lse)


def _exact_drafts(case, s):
    vocab, lists = case["vocab"], case["form"] == "lists"

    def dense(name, row):  # one row's probabilities by id, f64
        if not lists:
            return s[name][row].double()
        kept = int(s[name + "_kept"][row])
        return torch.zeros(vocab, dtype=torch.float64, device=DEV).index_add_(
            0, s[name + "_ids"][row, :kept].long(), s[name][row, :kept].double())

    accepted, tokens = [], []
    drafted, uniforms, draws = s["drafted"].tolist(), s["uniforms"].tolist(), s["draws"].tolist()
    starts = s["starts"].tolist()
    for i, n in enumerate(s["lens"].tolist()):
        a, said = starts[i], []
        for j in range(n + 1):
            p = dense("target", a + i + j)
            if j < n:
                d = drafted[a + j]
                q = dense("draft", a + j) if s["draft"] is not None else torch.zeros_like(p).index_fill_(
                    0, torch.tensor([d], device=DEV), 1.0)
                if uniforms[a + j] * float(q[d]) < float(p[d]):
                    said.append(d)
                    continue
                rest = torch.relu(p - q)
                p = rest if bool((rest > 0).any()) else p
            if lists:  # candidates are drawn in their own order
                ids = s["target_ids"][a + i + j, :int(s["target_kept"][a + i + j])].long()
                p = p[ids]
            border = torch.cumsum(p, 0)
            at = int(torch.searchsorted(border, border[-1:] * draws[i], right=True)[0])
            said.append(int(ids[at]) if lists else at)
            break
        accepted.append(len(said) - 1)
        tokens += said + [-1] * (n + 1 - len(said))
    return (torch.tensor(accepted, dtype=torch.int32, device=DEV), torch.tensor(tokens, dtype=torch.int32, device=DEV))
