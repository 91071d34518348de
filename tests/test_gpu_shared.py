"""Attention behind shared prefixes on the GPU: against the float64 statement of
attention (mixer_fixtures.py) over the prefix's and the sequence's own tokens in one, and
against rl_attention_rows over tables that hold both."""
import numpy as np
import pytest
import torch

import mixer_fixtures as F
import rl_mixers as M
import rl_sampler as R
from test_gpu_mixers import attend_check, paged, randn, strided

pytestmark = pytest.mark.gpu


def i32(x, device):
    return torch.from_numpy(np.ascontiguousarray(x, np.int32)).to(device)


class Case:
    def __init__(self, g, device, prefixes, per, lens, counts, qh, kv, dim, page, fmt, dtype, spread=2.0, fill=float("nan"),
                 max_len=None):
        """prefixes: tokens of each group's; per: its sequences."""
        self.__dict__.update(prefixes=prefixes, per=per, lens=lens, counts=counts, dim=dim, fmt=fmt, dtype=dtype)
        source = "f16" if fmt == "f16" else "bf16"
        both = list(prefixes) + list(lens)
        table, pages = paged(g, both, page)
        self.cache = M.DeviceCache(pages, page, kv, dim, fmt)
        rest = torch.full((pages * page, kv, dim), fill, device=device)
        self.cache.write(rest, rest, torch.arange(pages * page, device=device))
        held = []
        for i, n in enumerate(both):
            k, v = (randn(g, (n, kv, dim), source, device) for _ in range(2))
            t = np.arange(n)
            if n:
                self.cache.write(k, v, torch.from_numpy(table[i, t // page].astype(np.int64) * page + t % page).to(device))
            held.append((F.encode(F.as64(k), fmt), F.encode(F.as64(v), fmt)))
        m = len(prefixes)
        group = np.repeat(np.arange(m), per)
        self.stored = [tuple(np.concatenate([a, b]) for a, b in zip(held[group[i]], held[m + i])) for i in range(len(lens))]
        self.whole = [prefixes[group[i]] + n for i, n in enumerate(lens)]
        self.q = randn(g, (sum(counts), qh, dim), dtype, device, spread)
        self.out = torch.full_like(self.q, 7.0)
        self.lse = torch.full(self.q.shape[:2], 7.0, device=device)
        self.table, self.prefix_table = i32(table[m:], device), i32(table[:m], device)
        self.t = dict(lens=i32(lens, device), groups=i32(np.concatenate([[0], np.cumsum(per)]), device),
                      prefix_lens=i32(prefixes, device))
        self.starts = None if all(c == 1 for c in counts) else i32(np.concatenate([[0], np.cumsum(counts)]), device)
        self.att = M.DeviceAttention(max(sum(counts), 1), qh, kv, dim, max_len or max(both + [1]))

    def call(self, q=None, out=None, **kw):
        self.att.shared(self.cache, self.q if q is None else q, self.out if out is None else out, self.t["lens"], self.table,
                        self.t["groups"], self.t["prefix_lens"], self.prefix_table, starts=self.starts, lse=self.lse, **kw)
        torch.cuda.synchronize()

    def check(self, out=None, scale=None):
        """Rows that stand before their sequence's first token see the prefix alone."""
        at, out = 0, self.out if out is None else out
        for n, p, c, held in zip(self.lens, np.repeat(self.prefixes, self.per), self.counts, self.stored):
            early = max(c - n, 0)
            for i in range(early):
                attend_check(self.q[at + i:at + i + 1], out[at + i:at + i + 1], self.lse[at + i:at + i + 1], [p], [1],
                             [tuple(x[:p] for x in held)], self.fmt, self.dtype, 0, self.dim, scale)
            if c > early:
                attend_check(self.q[at + early:at + c], out[at + early:at + c], self.lse[at + early:at + c], [p + n], [c - early],
                             [held], self.fmt, self.dtype, 0, self.dim, scale)
            at += c


SHARED = [
    # prefixes, sequences of each, lens, rows, q heads, kv heads, dim, page, format, type
    ([1], [1], [1], [1], 1, 1, 16, 1, "bf16", "bf16"),
    ([300], [5], [5, 0, 64, 129, 17], [1] * 5, 8, 2, 128, 16, "bf16", "bf16"),
    ([777, 0, 130], [3, 2, 1], [5, 40, 64, 9, 100, 2], [1, 3, 2, 4, 1, 2], 8, 2, 128, 24, "i8", "bf16"),
    ([33, 500], [4, 4], [1, 2, 3, 0, 50, 60, 70, 80], [1] * 8, 12, 3, 80, 7, "f8", "f32"),
    ([2000], [7], [30, 40, 50, 60, 70, 80, 90], [5] * 7, 16, 4, 64, 32, "f16", "f16"),
    ([1500, 64], [2, 2], [2100, 3, 900, 40], [2, 2, 2, 2], 8, 2, 256, 24, "f16", "f32"),   # own tokens in several parts
    ([400], [3], [2, 1, 0], [5, 3, 2], 6, 1, 96, 40, "bf16", "f32"),     # rows before the first own token
    ([0, 0], [1, 2], [0, 5, 0], [1, 1, 1], 4, 2, 48, 16, "i8", "f16"),   # some see nothing at all
    ([4097], [40], [1 + i % 30 for i in range(40)], [1] * 40, 32, 4, 128, 64, "i8", "bf16"),
    ([1024, 1024, 1000], [20, 1, 0], [9] * 21, [4] * 21, 16, 2, 128, 16, "bf16", "bf16"),  # a group without sequences
    ([700], [64], [16] * 64, [1] * 64, 64, 1, 64, 48, "f8", "bf16"),
    ([513], [9], [11] * 9, [9] * 9, 5, 5, 112, 16, "bf16", "f32"),
    ([1300, 40], [30, 3], [7] * 33, [2] * 33, 12, 2, 112, 16, "bf16", "f32"),  # the three parts of f32 queries and weights
    ([900], [40], [3 + i for i in range(40)], [1] * 40, 8, 2, 256, 32, "f16", "f32"),
    ([2049], [20], [5] * 20, [3] * 20, 16, 4, 64, 24, "f8", "f32"),
    ([1025, 3000], [30, 40], [20] * 70, [1] * 70, 16, 2, 48, 48, "i8", "f16"),
    ([700], [50], [9] * 50, [1] * 50, 16, 4, 256, 7, "bf16", "bf16"),
    ([65, 64, 63, 1], [40, 40, 40, 40], [1 + i % 5 for i in range(160)], [1] * 160, 8, 2, 80, 16, "f16", "f16"),
    ([300], [31], [70] + [3] * 30, [60] + [1] * 30, 8, 2, 128, 16, "bf16", "bf16"),  # one sequence of many rows among single ones
    ([90, 31], [20, 20], [600] * 40, [1] * 40, 8, 2, 64, 16, "i8", "bf16"),  # more tokens of their own than shared ones
    # Too many workgroups for one launch, few rows of each group: joined by the sequence's own, in parts, two row tiles.
    ([100 + 7 * i for i in range(40)], [2] * 40, [1 + i for i in range(80)], [1] * 80, 8, 8, 64, 16, "bf16", "bf16"),
    ([50 + 3 * i for i in range(40)], [2] * 40, [150 + 3 * i for i in range(80)], [1] * 80, 8, 8, 128, 24, "i8", "f32"),
    ([500 - 9 * i for i in range(20)], [4] * 20, [2 + i for i in range(80)], [2] * 80, 32, 8, 64, 16, "f8", "f16"),
    ([200] * 20, [4] * 20, [30] * 80, [5] * 80, 16, 8, 48, 7, "f16", "f16"),
]


@pytest.mark.parametrize("case", range(len(SHARED)))
def test_shared(device, case):
    g = np.random.default_rng(400 + case)
    c = Case(g, device, *SHARED[case])
    print("shared", SHARED[case], flush=True)
    bounds = dict(most_rows=max(c.counts), max_len=max(max(c.lens), 1), max_prefix=max(max(c.prefixes), 1))
    c.call(**bounds)
    c.check()
    first, first_lse = c.out.clone(), c.lse.clone()
    c.call()  # without bounds
    c.check()
    c.out.fill_(3.0)
    c.call(**bounds)
    assert torch.equal(c.out, first) and torch.equal(c.lse, first_lse)  # no result depends on an order of arrival


def test_shared_as_rows_over_whole_tables(device):
    # Prefixes of whole pages: the table of a sequence is its prefix's pages and then its own.
    g = np.random.default_rng(21)
    c = Case(g, device, [96, 480], [3, 4], [5, 100, 40, 1, 2, 300, 77], [1, 2, 3, 1, 1, 2, 3], 8, 2, 128, 32, "i8", "bf16")
    c.call()
    tables = []
    for i, group in enumerate([0, 0, 0, 1, 1, 1, 1]):
        n = c.prefixes[group] // 32
        tables.append(np.concatenate([c.prefix_table[group, :n].cpu().numpy(), c.table[i].cpu().numpy()]))
    width = max(map(len, tables))
    whole = i32([np.pad(t, (0, width - len(t))) for t in tables], device)
    out, lse = torch.empty_like(c.out), torch.empty_like(c.lse)
    att = M.DeviceAttention(c.q.shape[0], 8, 2, 128, 800)
    att.rows(c.cache, c.q, out, i32(c.whole, device), whole, starts=c.starts, lse=lse)
    torch.cuda.synchronize()
    # Both are within a thousandth of the output's rounding of the exact value: bf16 values that differ are neighbours.
    a, b = F.as64(c.out), F.as64(out)
    assert np.all(np.abs(a - b) <= np.maximum(np.abs(a), np.abs(b)) * 2.0 ** -7 + 1e-6)
    assert np.abs(F.as64(c.lse) - F.as64(lse)).max() <= 1e-5


def test_shared_strides_and_large_scores(device):
    g = np.random.default_rng(22)
    for more in (1, 40):
        c = Case(g, device, [130, 77], [2 * more, 1], [30, 4] * more + [50], [2, 1] * more + [3], 4, 2, 64, 16, "bf16", "f32",
                 spread=60.0)
        for pads in ((0, 0), (1, 3), (8, 4)):
            qs, outs = strided(c.q, *pads, device), strided(c.out, *pads, device)
            for scale in (1.0, -0.5, 0.0):  # of another sign, and all weights alike
                c.call(qs, outs, scale=scale)
                c.check(outs, scale=scale)


@pytest.mark.parametrize("heads,own", [(4, 20), (64, 20), (4, 900)])  # few and many rows of a prefix; own tokens in parts
def test_shared_sequences_of_no_group_and_rows_behind_the_last(device, heads, own):
    g = np.random.default_rng(27)
    c = Case(g, device, [0, 300, 0], [2, 3, 2], [own, 5, own, 6, 3, 7, own], [2, 1, 1, 2, 3, 1, 2], heads, 2, 64, 16, "bf16", "bf16")
    c.call()  # every partial result and count of the handle has been used
    c.out.fill_(7.0)
    c.lse.fill_(7.0)
    c.t.update(groups=i32([2, 5], device), prefix_lens=i32([300], device))
    c.prefix_table = c.prefix_table[1:2].contiguous()
    c.call()
    c.check()
    # A batch that holds fewer rows than the call has: the others stay as they were.
    c.out.fill_(7.0)
    c.lse.fill_(7.0)
    c.starts[-1] = 10  # the last sequence has none
    c.call()
    assert (c.out[10:] == 7.0).all() and (c.lse[10:] == 7.0).all()
    c.lens, c.counts, c.per = c.lens[:-1], c.counts[:-1], [2, 3, 1]
    c.check()
    att = M.DeviceAttention(12, heads, 2, 64, 40000)
    table = c.table.expand(-1, -1)[:, :1].expand(-1, 2500).contiguous()  # the same page over and over
    lens = i32([40000] * 7, device)
    for n in (12, 10):
        c.out.fill_(7.0)
        c.starts[-1] = n
        att.rows(c.cache, c.q, c.out, lens, table, starts=c.starts, lse=c.lse)
        torch.cuda.synchronize()
        assert (c.out[n:] == 7.0).all() and (c.out[:n] != 7.0).any((1, 2)).all()


@pytest.mark.parametrize("heads", [4, 128])  # few rows and heads of a prefix, and many
def test_shared_past_its_bounds_gives_nan(device, heads):
    g = np.random.default_rng(23)
    spec = ([200, 60, 90], [2, 1, 2], [10, 20, 30, 40, 50], [1] * 5, heads, 2, 32, 16, "i8", "bf16")

    def nan_rows(rows):
        got = np.isnan(F.as64(c.out)).all((1, 2)) & np.isnan(F.as64(c.lse)).all(1)
        assert np.array_equal(np.flatnonzero(got), rows), got
        assert not np.isnan(F.as64(c.out)[[i for i in range(5) if i not in rows]]).any()

    c = Case(g, device, *spec)
    c.call(max_prefix=199)
    nan_rows([0, 1])
    c.call(max_len=45)
    nan_rows([4])
    c.t["prefix_lens"][0] = 2 ** 31 - 1
    c.call()
    nan_rows([0, 1])
    c = Case(g, device, *spec)
    c.t["prefix_lens"][0] = -5  # as none: the rows see their own tokens
    c.call()
    nan_rows([])
    attend_check(c.q[:1], c.out[:1], c.lse[:1], [10], [1], [tuple(x[200:] for x in c.stored[0])], "i8", "bf16", 0, 32)
    c.prefix_table[1, 3] = 10 ** 6  # no page of the cache
    c.table[3, 0] = -1
    c.call()
    nan_rows([2, 3])
    c = Case(g, device, *spec)
    c.prefix_table = c.prefix_table[:, :5].contiguous()  # 200 tokens need 13 pages, 90 need 6
    c.call()
    nan_rows([0, 1, 3, 4])


def test_shared_values_out_of_sight(device):
    # Own tokens past a row's, and what stands in the pages' rest, are NaN (fill) or infinite: they reach no row.
    g = np.random.default_rng(24)
    for fmt, dtype in (("bf16", "bf16"), ("f16", "f32"), ("f8", "bf16"), ("i8", "f32")):
        for more in (1, 40):  # few rows of a prefix, and many
            c = Case(g, device, [50, 21], [2 * more, 2], [3, 30] * more + [17, 1], [2, 3] * more + [1, 1], 4, 2, 64, 16, fmt,
                     dtype, fill=float("inf"))
            c.call()
            c.check()


def test_shared_scores_of_minus_infinity(device):
    # Tokens that are seen with a score of -inf have no weight beside others, and a row that sees only such is NaN, as
    # elsewhere; so is none that sees a finite score.
    cache = M.DeviceCache(4, 16, 1, 16, "bf16")
    k, v = torch.zeros(64, 1, 16, device=device), torch.ones(64, 1, 16, device=device)
    k[:16, 0, 0] = -float("inf")  # page 0
    cache.write(k, v, torch.arange(64, device=device))
    q = torch.ones(2, 1, 16, device=device, dtype=torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty(2, 1, device=device)
    att = M.DeviceAttention(2, 1, 1, 16, 64)
    for own, prefix, want in ((1, 0, 1.0), (0, 1, 1.0), (0, 0, float("nan"))):
        att.shared(cache, q, out, i32([4, 16], device), i32([[own], [own]], device), i32([0, 2], device), i32([16], device),
                   i32([[prefix]], device), lse=lse)
        torch.cuda.synchronize()
        got = F.as64(out)
        assert np.isnan(got).all() if want != want else (got == want).all(), (own, prefix, got)


def test_shared_captured_and_another_stream(device):
    g = np.random.default_rng(25)
    for spec in (SHARED[2], SHARED[5]):
        c = Case(g, device, *spec)
        c.call()
        want, want_lse = c.out.clone(), c.lse.clone()
        other = torch.cuda.Stream()
        c.out.zero_()
        torch.cuda.synchronize()
        c.call(stream=other.cuda_stream)
        assert torch.equal(c.out, want)
        graph = torch.cuda.CUDAGraph()
        args = (c.cache, c.q, c.out, c.t["lens"], c.table, c.t["groups"], c.t["prefix_lens"], c.prefix_table)
        with torch.cuda.graph(graph):
            c.att.shared(*args, starts=c.starts, lse=c.lse)
        for i in range(4):
            c.q.mul_(-1.0)  # other inputs, and the handle used by an eager call between the replays
            c.call()
            want, want_lse = c.out.clone(), c.lse.clone()
            c.out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(c.out, want) and torch.equal(c.lse, want_lse)


def test_shared_refusals(device):
    g = np.random.default_rng(26)
    c = Case(g, device, [40], [2], [3, 4], [1, 1], 4, 2, 32, 16, "bf16", "bf16")

    def refused(code, **kw):
        with pytest.raises(R.SamplerError) as e:
            c.call(**kw)
        assert e.value.code == code

    refused(R.RL_ERR_CAPACITY, max_prefix=41)
    refused(R.RL_ERR_CAPACITY, max_len=41)
    c.t["groups"], c.t["prefix_lens"] = i32([0, 1, 1, 2], device), i32([4, 4, 4], device)
    c.prefix_table = c.prefix_table.expand(3, -1).contiguous()
    refused(R.RL_ERR_ARGUMENT)  # more groups than sequences
