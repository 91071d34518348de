"""What is timed of the token mixers: the calls that a decode step, a speculative
verify, a serving batch and a prompt make between the embedding lookup and the
output head.

  rotary   rotary positions of the query and key heads, one call for both
  cache    keys (rotated) and values written into a paged cache, then read back
  attend   attention of new tokens over the paged cache
  delta    the gated delta rule: one step of a batch, a verify, prompts

The plain forms are elementary torch operations in f32, rounded once to the
output's type. Sequence lengths follow from the case alone; their order, the
pages' order and all values follow from the seed. The states of `delta` are read
from one half of a pool and written to the other, as a program does that may
have to go back to the state before a verify, so a pass can be repeated.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
WIDTH = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1, "f8": 1}
EPS = 1e-6


def _rotary(name, rows, q_heads, k_heads, dim, turned, layout, dtype, scaling="none", context=32768, inverse=False):
    return {"name": name, "op": "rotary", "rows": rows, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "turned": turned, "layout": layout, "dtype": dtype, "scaling": scaling, "context": context,
            "inverse": inverse}


def _cache(name, rows, heads, dim, page, fmt, dtype, turned, layout, context=32768):
    return {"name": name, "op": "cache", "rows": rows, "heads": heads, "dim": dim, "page": page, "format": fmt,
            "dtype": dtype, "turned": turned, "layout": layout, "context": context}


def _attend(name, seqs, shortest, longest, rows, q_heads, kv_heads, dim, page, fmt, dtype, window=0):
    return {"name": name, "op": "attend", "seqs": seqs, "shortest": shortest, "longest": longest, "rows": rows,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "format": fmt, "dtype": dtype,
            "window": window}


def _delta(name, seqs, shortest, longest, key_heads, value_heads, key_dim, value_dim, dtype, normalise=True):
    return {"name": name, "op": "delta", "seqs": seqs, "shortest": shortest, "longest": longest,
            "key_heads": key_heads, "value_heads": value_heads, "key_dim": key_dim, "value_dim": value_dim,
            "dtype": dtype, "normalise": normalise}


def listed():
    return [
        # One token of one sequence, a quarter of each head turned: all launch
        # and latency.
        _rotary("rotary_1", 1, 16, 4, 256, 64, "half", "bf16"),
        # A prompt in the f32 rows that the embedding lookup gives, whole heads
        # turned, frequencies stretched for a long context: the largest call.
        _rotary("rotary_4096", 4096, 32, 8, 128, 128, "interleaved", "f32", scaling="yarn", context=131072),
        # The step of a serving batch: a token a sequence into an int8 cache.
        _cache("cache_64", 64, 8, 128, 32, "i8", "bf16", 128, "half"),
        # A prompt of odd length into an 8-bit float cache.
        _cache("cache_5003", 5003, 4, 256, 64, "f8", "bf16", 64, "half"),
        # One token of one sequence after a short prompt: the smallest call.
        _attend("attend_short", 1, 611, 611, 1, 16, 4, 256, 32, "bf16", "bf16"),
        # One token of one sequence at a long context: the cache's length has to
        # be shared out.
        _attend("attend_long", 1, 131071, 131071, 1, 32, 8, 128, 64, "bf16", "bf16"),
        # The step of a serving batch whose sequences differ 64-fold in length,
        # over an int8 cache.
        _attend("attend_batch_64", 64, 128, 8192, 1, 32, 8, 128, 32, "i8", "bf16"),
        # The check of eight drafted tokens with f32 queries, pages of 24 tokens
        # (they end inside any tile).
        _attend("attend_verify_9", 1, 20011, 20011, 9, 16, 4, 256, 24, "f16", "f32"),
        # The step of a serving batch: states in and out, one token each.
        _delta("delta_64", 64, 1, 1, 16, 32, 128, 128, "bf16"),
        # The check of eight drafted tokens of one sequence.
        _delta("delta_verify_9", 1, 9, 9, 16, 32, 128, 128, "bf16"),
        # A long prompt of one sequence.
        _delta("delta_prompt_8192", 1, 8192, 8192, 16, 32, 128, 128, "bf16"),
        # A few prompts of odd lengths in f32.
        _delta("delta_ragged_7", 7, 33, 701, 8, 8, 64, 96, "f32", normalise=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "cache", "attend", "attend", "delta", "delta"])
    dim = rng.choice([64, 80, 96, 128, 256])
    layout = rng.choice(["half", "interleaved"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    turned = rng.choice([dim, dim, dim // 2, dim // 4])
    if op == "rotary":
        c = _rotary("", _log_int(rng, 1, 4096), rng.choice([8, 12, 16, 32]), rng.choice([1, 2, 4, 8]), min(dim, 128),
                    min(turned, 128), layout, dtype, rng.choice(["none", "linear", "yarn"]),
                    rng.choice([4096, 32768, 131072]), rng.random() < 0.3)
    elif op == "cache":
        c = _cache("", _log_int(rng, 1, 8192), rng.choice([1, 2, 4, 8]), dim, rng.choice([16, 24, 32, 64]),
                   rng.choice(["i8", "f8", "i8", "f8", "bf16", "f16"]), dtype, turned, layout)
    elif op == "attend":
        seqs, kv_heads, rows = _log_int(rng, 1, 96), rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 1, 2, 5, 9])
        # At most the longest listed case's keys and values.
        longest = _log_int(rng, 16, min(65536, (1 << 27) // (seqs * kv_heads * dim)))
        shortest = max(1, longest // rng.choice([1, 4, 64]))
        fmt = rng.choice(["i8", "f8", "i8", "f8", "same", "same"])
        fmt = ("f16" if dtype == "f16" else "bf16") if fmt == "same" else fmt
        window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        c = _attend("", seqs, max(rows, shortest), max(rows, longest), rows, kv_heads * rng.choice([1, 2, 4, 8] if rows <= 2 else [1, 2, 4]),
                    kv_heads, dim, rng.choice([16, 24, 32, 64, 128]), fmt, dtype, window)
    else:
        key_heads = rng.choice([2, 4, 8, 16])
        kind = rng.choice(["step", "verify", "prompt", "prompt"])
        seqs = _log_int(rng, 1, 96) if kind == "step" else _log_int(rng, 1, 12)
        longest = {"step": 1, "verify": rng.choice([2, 5, 9, 17]), "prompt": _log_int(rng, 32, 8192 // seqs)}[kind]
        shortest = max(1, longest // rng.choice([1, 2, 16])) if kind == "prompt" else longest
        c = _delta("", seqs, shortest, longest, key_heads, key_heads * rng.choice([1, 2]), rng.choice([64, 96, 128]),
                   rng.choice([64, 96, 128]), dtype, rng.random() < 0.7)
    del c["name"]
    return c


def _spread(case):
    # Lengths from the shortest to the longest, evenly over their logarithm.
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    return [int(round(a * (b / a) ** (i / (n - 1)))) for i in range(n)] if n > 1 else [b]


def work(case):
    op = case["op"]
    if op == "rotary":
        values = case["rows"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        return {"bytes": 2 * values * WIDTH[case["dtype"]] + 8 * case["rows"],
                "flops": 3 * values * case["turned"] / case["dim"]}
    if op == "cache":
        vectors = 2 * case["rows"] * case["heads"]
        code = case["dim"] * WIDTH[case["format"]] + (4 if WIDTH[case["format"]] == 1 else 0)
        return {"bytes": vectors * (case["dim"] * (WIDTH[case["dtype"]] + 2) + 2 * code) + 24 * case["rows"],
                "flops": 6 * vectors * case["dim"]}
    if op == "attend":
        lens = _spread(case)
        seen = [min(n, case["window"] + case["rows"] - 1) if case["window"] else n for n in lens]
        code = case["dim"] * WIDTH[case["format"]] + (4 if WIDTH[case["format"]] == 1 else 0)
        heads = case["seqs"] * case["rows"] * case["q_heads"]
        return {"bytes": sum(seen) * case["kv_heads"] * 2 * code + 2 * heads * case["dim"] * WIDTH[case["dtype"]],
                "flops": 4 * sum(seen) * case["rows"] * case["q_heads"] * case["dim"]}
    rows, dk, dv, size = sum(_spread(case)), case["key_dim"], case["value_dim"], WIDTH[case["dtype"]]
    return {"bytes": rows * (2 * case["key_heads"] * dk * size + case["value_heads"] * (2 * dv * size + 8))
            + case["seqs"] * case["value_heads"] * dk * dv * 8,
            "flops": 6 * rows * case["value_heads"] * dk * dv}


# ---------------------------------------------------------------- inputs --
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * sigma).to(TYPES[dtype])


def _frequencies(case):
    """Radians a position of each pair, f64, and the magnitude of the result."""
    d, base, factor, original = case["turned"], 1e6, 4.0, case["context"] // 4
    f = base ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    scaling = case.get("scaling", "none")
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        def place(turns):
            return d * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), d - 1)
        ramp = ((torch.arange(d // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1
    return f, 1.0


def _inputs(case, seed):
    """The tensors that both forms start from."""
    g, op = _generator(seed), case["op"]
    if op == "rotary":
        s = {"q": _normal(g, (case["rows"], case["q_heads"], case["dim"]), case["dtype"]),
             "k": _normal(g, (case["rows"], case["k_heads"], case["dim"]), case["dtype"])}
        # A prompt's positions follow one another from anywhere in the context.
        at = torch.randint(0, case["context"] - case["rows"] + 1, (1,), generator=g, device=DEV)
        s["positions"] = at + torch.arange(case["rows"], device=DEV)
        return s
    if op == "cache":
        shape, rows, page = (case["rows"], case["heads"], case["dim"]), case["rows"], case["page"]
        # Keys have a few channels far larger than the rest, values have not.
        channel = 1 + 7 * (torch.rand(case["heads"], case["dim"], generator=g, device=DEV) < 0.03)
        s = {"k": (torch.randn(shape, generator=g, device=DEV) * channel).to(TYPES[case["dtype"]]),
             "v": _normal(g, shape, case["dtype"], 0.5)}
        pages = rows if rows <= 128 else -(-rows // page) + 3
        order = torch.randperm(pages, generator=g, device=DEV)
        if rows <= 128:  # one token a sequence, each in a page of its own
            s["slots"] = order[:rows] * page + torch.randint(0, page, (rows,), generator=g, device=DEV)
            s["positions"] = torch.randint(0, case["context"], (rows,), generator=g, device=DEV)
        else:  # a prompt
            t = torch.arange(rows, device=DEV)
            s["slots"] = order[t // page] * page + t % page
            s["positions"] = t
        s["pages"] = pages
        return s
    if op == "attend":
        lens = torch.tensor(_spread(case), device=DEV)[torch.randperm(case["seqs"], generator=g, device=DEV)]
        page, longest = case["page"], case["longest"]
        width = -(-longest // page)
        need = -(-lens // page)
        pages = sum(-(-n // page) for n in _spread(case))
        order = torch.randperm(pages, generator=g, device=DEV)
        first = torch.cumsum(need, 0) - need
        j = torch.arange(width, device=DEV)
        at = (first[:, None] + j).clamp(max=pages - 1)
        table = torch.where(j < need[:, None], order[at], torch.zeros_like(at))
        source = "f16" if case["format"] == "f16" else "bf16"
        shape = (pages * page, case["kv_heads"], case["dim"])
        return {"k": _normal(g, shape, source), "v": _normal(g, shape, source),
                "q": _normal(g, (case["seqs"] * case["rows"], case["q_heads"], case["dim"]), case["dtype"], 2.0),
                "lens": lens.to(torch.int32), "table": table.to(torch.int32), "pages": pages}
    lens = torch.tensor(_spread(case), device=DEV)[torch.randperm(case["seqs"], generator=g, device=DEV)]
    rows, kh, vh = sum(_spread(case)), case["key_heads"], case["value_heads"]
    unit = 1.0 if case["normalise"] else case["key_dim"] ** -0.5
    k = torch.randn((rows, kh, case["key_dim"]), generator=g, device=DEV)
    k = k if case["normalise"] else k / k.square().sum(-1, keepdim=True).sqrt()
    return {"q": _normal(g, (rows, kh, case["key_dim"]), case["dtype"], unit), "k": k.to(TYPES[case["dtype"]]),
            "v": _normal(g, (rows, vh, case["value_dim"]), case["dtype"]),
            # Decays from 0.998 to under a half a token, by head.
            "g": -torch.exp(torch.linspace(-6.0, 0.0, vh, device=DEV)
                            + 0.5 * torch.randn((rows, vh), generator=g, device=DEV)),
            "beta": torch.sigmoid(torch.randn((rows, vh), generator=g, device=DEV)),
            "states": 0.3 * torch.randn((2 * case["seqs"], vh, case["key_dim"], case["value_dim"]), generator=g,
                                        device=DEV),
            "lens": lens,
            "starts": torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(lens, 0)]).to(torch.int32)}


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


def _decode(codes, scale):
    x = codes.to(torch.float32)
    return x if scale is None else x * scale


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"], op = case, case["op"]
    if own:
        return _prepare_own(s, case)
    if "turned" in case:  # cosines and sines of every position of the context
        f, magnitude = _frequencies(case)
        angle = torch.arange(case["context"], dtype=torch.float64, device=DEV)[:, None] * f.to(DEV)
        s["cos"], s["sin"] = (magnitude * angle.cos()).float(), (magnitude * angle.sin()).float()
    if op == "cache":
        empty = torch.zeros((s["pages"] * case["page"], case["heads"], case["dim"]), device=DEV)
        s["pool_k"], s["pool_v"] = _encode(empty, case["format"]), _encode(empty, case["format"])
    if op == "attend":
        s["pool_k"], s["pool_v"] = _encode(s["k"].float(), case["format"]), _encode(s["v"].float(), case["format"])
        del s["k"], s["v"]
    return s


def _prepare_own(s, case):
    sys.path.insert(0, os.path.abspath("rust-llm_amd"))
    import rl_mixers
    op = case["op"]
    if "turned" in case:
        s["rotary"] = rl_mixers.DeviceRotary(case["turned"], base=1e6, layout=case["layout"],
                                             scaling=case.get("scaling", "none"), factor=4.0,
                                             original=case["context"] // 4)
    if op == "rotary":
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    elif op == "cache":
        s["cache"] = rl_mixers.DeviceCache(s["pages"], case["page"], case["heads"], case["dim"], case["format"])
        s["k_out"] = torch.empty(s["k"].shape, dtype=torch.bfloat16, device=DEV)
        s["v_out"] = torch.empty_like(s["k_out"])
    elif op == "attend":
        s["cache"] = rl_mixers.DeviceCache(s["pages"], case["page"], case["kv_heads"], case["dim"], case["format"])
        s["cache"].write(s["k"], s["v"], torch.arange(s["k"].shape[0], device=DEV))
        del s["k"], s["v"]
        s["attention"] = rl_mixers.DeviceAttention(s["q"].shape[0], case["q_heads"], case["kv_heads"], case["dim"],
                                                   case["longest"])
        s["starts"] = torch.arange(case["seqs"] + 1, dtype=torch.int32, device=DEV) * case["rows"]
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=DEV)
    else:
        s["delta"] = rl_mixers.DeviceDelta(s["q"].shape[0], case["seqs"], case["key_heads"], case["value_heads"],
                                           case["key_dim"], case["value_dim"])
        slots = torch.arange(2 * case["seqs"], dtype=torch.int32, device=DEV)
        s["before"], s["after"] = slots[:case["seqs"]], slots[case["seqs"]:]
        s["states_after"] = s["states"][case["seqs"]:]
        s["out"] = torch.empty_like(s["v"])
    return s


# ------------------------------------------------------------- the passes --
def run(s):
    op = s["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "cache": _own_cache, "attend": _own_attend, "delta": _own_delta}[op](s)
    return {"rotary": _plain_rotary, "cache": _plain_cache, "attend": _plain_attend, "delta": _plain_delta}[op](s)


def _own_rotary(s):
    s["rotary"].apply(s["q"], s["positions"], s["q_out"], second=s["k"], second_out=s["k_out"],
                      inverse=s["case"]["inverse"])
    return s["q_out"], s["k_out"]


def _own_cache(s):
    s["cache"].write(s["k"], s["v"], s["slots"], rotary=s["rotary"], positions=s["positions"])
    s["cache"].read(s["slots"], s["k_out"], s["v_out"])
    return s["k_out"], s["v_out"]


def _own_attend(s):
    c = s["case"]
    s["attention"].rows(s["cache"], s["q"], s["out"], s["lens"], s["table"], starts=s["starts"], lse=s["lse"],
                        window=c["window"], most_rows=c["rows"])
    return s["out"], s["lse"]


def _own_delta(s):
    s["delta"].rows(s["q"], s["k"], s["v"], s["g"], s["beta"], s["out"], s["states"], s["before"], s["after"],
                    s["starts"], normalise=s["case"]["normalise"], most_rows=s["case"]["longest"])
    return s["out"], s["states_after"]


def _turn(x, cos, sin, layout):
    """x [rows][heads][dim] f32 with its first pairs turned; cos, sin [rows][pairs]."""
    n = cos.shape[1]
    head, rest = x[..., :2 * n], x[..., 2 * n:]
    a, b = (head[..., :n], head[..., n:]) if layout == "half" else (head[..., 0::2], head[..., 1::2])
    cos, sin = cos[:, None], sin[:, None]
    a, b = a * cos - b * sin, a * sin + b * cos
    head = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([head, rest], -1)


def _plain_rotary(s):
    c = s["case"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    sin = -sin if c["inverse"] else sin
    return tuple(_turn(s[x].float(), cos, sin, c["layout"]).to(s[x].dtype) for x in ("q", "k"))


def _plain_cache(s):
    c, slots = s["case"], s["slots"]
    k = _turn(s["k"].float(), s["cos"][s["positions"]], s["sin"][s["positions"]], c["layout"])
    out = []
    for x, (codes, scale) in ((k, s["pool_k"]), (s["v"].float(), s["pool_v"])):
        new, new_scale = _encode(x, c["format"])
        if scale is None:
            codes[slots] = new
            out.append(codes[slots].to(torch.bfloat16))
        else:  # by bytes: indexing takes no 8-bit floats
            codes.view(torch.int8)[slots] = new.view(torch.int8)
            scale[slots] = new_scale
            out.append(_decode(codes.view(torch.int8)[slots].view(codes.dtype), scale[slots]).to(torch.bfloat16))
    return tuple(out)


def _plain_attend(s):
    c = s["case"]
    n, r, kv, page = c["seqs"], c["rows"], c["kv_heads"], c["page"]
    group = c["q_heads"] // kv
    t = torch.arange(c["longest"], device=DEV)
    slots = s["table"].long()[:, t // page] * page + t % page  # [seqs][longest]

    def gathered(pool):  # [seqs][kv heads][longest][dim]
        codes, scale = pool
        x = codes.view(torch.int8)[slots].view(codes.dtype) if codes.element_size() == 1 else codes[slots]
        return _decode(x, None if scale is None else scale[slots]).transpose(1, 2)

    q = s["q"].float().view(n, r, kv, group, c["dim"]).permute(0, 2, 1, 3, 4).reshape(n, kv, r * group, c["dim"])
    x = torch.matmul(q, gathered(s["pool_k"]).transpose(2, 3).contiguous()) * c["dim"] ** -0.5
    at = s["lens"].long()[:, None] - r + torch.arange(r, device=DEV)  # [seqs][rows]
    seen = t <= at[..., None]
    if c["window"]:
        seen &= t > at[..., None] - c["window"]
    x = x.masked_fill(~seen[:, None, :, None, :].expand(n, 1, r, group, -1).reshape(n, 1, r * group, -1), -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - top).exp()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, gathered(s["pool_v"]).contiguous()) / total
    def rows_first(y):
        return y.view(n, kv, r, group, -1).permute(0, 2, 1, 3, 4).reshape(n * r, c["q_heads"], -1)
    return rows_first(o).to(s["q"].dtype), rows_first(top + total.log())[..., 0].contiguous()


def _plain_delta(s):
    """Chunks of up to 64 tokens: within a chunk the corrected values solve a
    unit lower triangular system; the state passes from chunk to chunk."""
    c = s["case"]
    n, vh, dk, dv = c["seqs"], c["value_heads"], c["key_dim"], c["value_dim"]
    size = min(64, c["longest"])
    chunks = -(-c["longest"] // size)
    t = torch.arange(chunks * size, device=DEV)
    here = t < s["lens"][:, None]  # [seqs][tokens]
    at = (s["starts"][:-1].long()[:, None] + t).clamp(max=s["q"].shape[0] - 1)

    def chunked(x):  # [seqs][value heads][chunks][size][...], zero past a sequence's end
        x = x.float()[at] * here.view(n, -1, *[1] * (x.dim() - 1))
        return x.view(n, chunks, size, *x.shape[2:]).movedim(3, 1)

    def unit(x):
        return x / (x.square().sum(-1, keepdim=True) + EPS).sqrt() if c["normalise"] else x

    q, k = (unit(chunked(s[x])).repeat_interleave(vh // c["key_heads"], 1) for x in ("q", "k"))
    q = q * dk ** -0.5
    v, g, beta = chunked(s["v"]), chunked(s["g"]).cumsum(-1), chunked(s["beta"])[..., None]
    i = torch.arange(size, device=DEV)
    decay = (g[..., :, None] - g[..., None, :]).masked_fill(i[:, None] < i, -math.inf).exp()
    kt = k.transpose(-1, -2).contiguous()
    low = (torch.matmul(k, kt) * beta * decay).masked_fill(i[:, None] == i, 0.0)
    inverse = torch.eye(size, device=DEV).expand_as(low).clone()
    for j in range(1, size):  # row by row: inverse = (1 + low)^-1
        inverse[..., j, :j] = -torch.matmul(low[..., j:j + 1, :j], inverse[..., :j, :j])[..., 0, :]
    from_v = torch.matmul(inverse, beta * v)
    from_state = torch.matmul(inverse, beta * g.exp()[..., None] * k)
    within = torch.matmul(q, kt) * decay
    q = q * g.exp()[..., None]
    last = g[..., -1:]
    kt = (k * (last - g).exp()[..., None]).transpose(-1, -2).contiguous()
    state, out = s["states"][:n], torch.empty_like(v)
    for j in range(chunks):
        u = from_v[:, :, j] - torch.matmul(from_state[:, :, j], state)
        out[:, :, j] = torch.matmul(q[:, :, j], state) + torch.matmul(within[:, :, j], u)
        state = state * last[:, :, j, :, None].exp() + torch.matmul(kt[:, :, j], u)
    out = out.movedim(1, 3).reshape(n, chunks * size, vh, dv)
    return out[here].to(s["v"].dtype), state


# ------------------------------------------------------ the same in 64 bits --
def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotary": _exact_rotary, "cache": _exact_cache, "attend": _exact_attend, "delta": _exact_delta}[case["op"]](case, s)


def _exact_turn(case, x, positions, sign=1.0):
    f, magnitude = _frequencies(case)
    z = torch.polar(torch.full((1,), magnitude, dtype=torch.float64, device=DEV),
                    sign * positions.double()[:, None] * f.to(DEV))[:, None]  # [rows][1][pairs]
    y, n = x.double().clone(), case["turned"]
    first, second = (slice(0, n // 2), slice(n // 2, n)) if case["layout"] == "half" else (slice(0, n, 2), slice(1, n, 2))
    w = torch.complex(y[..., first], y[..., second]) * z
    y[..., first], y[..., second] = w.real, w.imag
    return y


def _exact_rotary(case, s):
    sign = -1.0 if case["inverse"] else 1.0
    return tuple(_exact_turn(case, s[x], s["positions"], sign) for x in ("q", "k"))


def _exact_stored(x, fmt):
    """What a cache of this format holds for f64 vectors. The step and the
    quotient that is rounded to a code are f32 by definition: halves occur."""
    if fmt in TYPES:
        return x.to(TYPES[fmt]).double()
    step = (x.abs().amax(-1, keepdim=True).float().double() / (127 if fmt == "i8" else 448)).float().double()
    y = (x.float().double() / torch.where(step > 0, step, 1.0)).float()
    return step * (y.double().round() if fmt == "i8" else y.to(torch.float8_e4m3fn).double())


def _exact_cache(case, s):
    return (_exact_stored(_exact_turn(case, s["k"], s["positions"]), case["format"]),
            _exact_stored(s["v"].double(), case["format"]))


def _exact_attend(case, s):
    r, page, kv = case["rows"], case["page"], case["kv_heads"]
    out, lse = [], []
    for i, n in enumerate(s["lens"].tolist()):
        t = torch.arange(n, device=DEV)
        slots = s["table"][i].long()[t // page] * page + t % page
        k, v = (_exact_stored(s[x][slots].double(), case["format"]).movedim(1, 0) for x in ("k", "v"))  # [kv][n][dim]
        q = s["q"][i * r:(i + 1) * r].double().view(r, kv, -1, case["dim"]).movedim(1, 0).flatten(1, 2)  # [kv][r group][dim]
        x = q @ k.transpose(1, 2) / math.sqrt(case["dim"])
        at = (n - r + torch.arange(r, device=DEV)).repeat_interleave(case["q_heads"] // kv)[:, None]
        x[:, (t > at) | ((t <= at - case["window"]) if case["window"] else False)] = -math.inf
        out.append((torch.softmax(x, -1) @ v).unflatten(1, (r, -1)).movedim(0, 1).flatten(1, 2))
        lse.append(torch.logsumexp(x, -1).unflatten(1, (r, -1)).movedim(0, 1).flatten(1, 2))
    return torch.cat(out), torch.cat(lse)


def _exact_delta(case, s):
    n, share = case["seqs"], case["value_heads"] // case["key_heads"]
    q, k, v = (s[x].double() for x in ("q", "k", "v"))
    if case["normalise"]:
        q, k = (x * torch.rsqrt((x * x).sum(-1, keepdim=True) + EPS) for x in (q, k))
    q, k = (x.repeat_interleave(share, 1) for x in (q / math.sqrt(case["key_dim"]), k))
    keep, beta = s["g"].double().exp()[..., None, None], s["beta"].double()[..., None]
    out, state = torch.zeros_like(v), s["states"][:n].double()
    starts, lens = s["starts"][:-1].tolist(), s["lens"].tolist()
    order = sorted(range(n), key=lambda i: -lens[i])  # the longest first: those still running lead
    state, first = state[order], torch.tensor([starts[i] for i in order], device=DEV)
    for t in range(max(lens)):
        m = sum(1 for i in lens if i > t)
        at = first[:m] + t
        a = keep[at] * state[:m]
        u = beta[at] * (v[at] - (k[at].unsqueeze(-2) @ a).squeeze(-2))
        a = a + k[at].unsqueeze(-1) * u.unsqueeze(-2)
        out[at] = (q[at].unsqueeze(-2) @ a).squeeze(-2)
        state[:m] = a
    back = torch.empty_like(state)
    back[order] = state
    return out, back
