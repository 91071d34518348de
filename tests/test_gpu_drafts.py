"""The verification of drafted tokens on the GPU against its float64 statement
(step_fixtures.py). What comes out are whole numbers: no input lies within rounding of a
border (uniforms have 24 bits, sums are f64), so they are equal."""
import numpy as np
import pytest
import torch

import rl_drafts as D
import rl_sampler as R
import step_fixtures as S

pytestmark = pytest.mark.gpu


def probs(g, rows, vocab, sharp):
    x = g.standard_normal((rows, vocab)) * sharp
    p = np.exp(x - x.max(1, keepdims=True))
    return (p / p.sum(1, keepdims=True)).astype(np.float32)


def dev(x, device):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(device)


def check(device, lens, target, draft, drafted, uniforms, draws, vocab, ids=None, kept=None, q_ids=None, q_kept=None,
          stride=None):
    """One call; target [drafts + seqs][..] and so on are numpy arrays."""
    n, starts = len(lens), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    handle = D.DeviceDrafts(n + 3, vocab)
    accepted = torch.full((n,), 77, dtype=torch.int32, device=device)
    tokens = torch.full((sum(lens) + n,), 77, dtype=torch.int32, device=device)

    def laid(p):
        if p is None or stride is None:
            return dev(p, device)
        buf = torch.full((p.shape[0], stride), float("nan"), device=device)
        buf[:, :p.shape[1]] = dev(p, device)
        return buf[:, :p.shape[1]]

    call = lambda: handle.verify(laid(target), dev(drafted.astype(np.int32), device), dev(starts, device),  # noqa: E731
                                 dev(uniforms.astype(np.float32), device), dev(draws.astype(np.float32), device), accepted,
                                 tokens, draft=laid(draft), target_ids=dev(ids, device), target_kept=dev(kept, device),
                                 draft_ids=dev(q_ids, device), draft_kept=dev(q_kept, device))
    call()
    torch.cuda.synchronize()

    def row(p, i, k, r):
        return (np.arange(vocab), p[r]) if i is None else (i[r, :min(k[r], p.shape[1])], p[r, :min(k[r], p.shape[1])])

    want_accepted, want_tokens = [], []
    for s, c in enumerate(lens):
        a = starts[s]
        rows = [row(target, ids, kept, r) for r in range(a + s, a + s + c + 1)]
        others = None if draft is None else [row(draft, q_ids, q_kept, r) for r in range(a, a + c)]
        k, t = S.verify(rows, others, drafted[a:a + c], uniforms.astype(np.float32)[a:a + c], np.float32(draws[s]))
        want_accepted.append(k)
        want_tokens += t
    assert accepted.tolist() == want_accepted
    assert tokens.tolist() == want_tokens
    call()
    torch.cuda.synchronize()
    assert tokens.tolist() == want_tokens
    handle.close()
    return want_accepted, want_tokens


DENSE = [
    # drafts of each, vocabulary, stride, form
    ([8], 151936, None, "dense"),
    ([0, 1, 5, 2, 0, 3], 1000, None, "dense"),
    ([4, 4], 4096, 4100, "dense"),
    ([3, 70, 200], 333, 335, "dense"),     # more drafts than a wave, unaligned rows
    ([2, 2, 2], 12289, 12292, "dense"),    # a last chunk of one token
    ([1] * 40, 8192, None, "greedy"),
    ([3, 0, 6], 5003, None, "greedy"),
    ([0, 0], 50000, None, "dense"),        # no drafts at all: two draws
    ([1, 2], 1, None, "dense"),
]


@pytest.mark.parametrize("sharp", [0.5, 3.0])
@pytest.mark.parametrize("case", range(len(DENSE)))
def test_dense_rows(device, case, sharp):
    lens, vocab, stride, form = DENSE[case]
    g = np.random.default_rng(case)
    drafts, n = sum(lens), len(lens)
    target = probs(g, drafts + n, vocab, sharp)
    row = np.concatenate([np.arange(c) + sum(lens[:s]) + s for s, c in enumerate(lens)]).astype(int) if drafts else np.zeros(0, int)
    mixed = 0.6 * target[row] + 0.4 * probs(g, drafts, vocab, sharp) if drafts else np.zeros((0, vocab))
    draft = mixed.astype(np.float32)
    drafted = np.array([g.choice(vocab, p=q / q.sum()) for q in draft.astype(np.float64)], np.int64)
    print("drafts", DENSE[case], sharp, flush=True)
    check(device, lens, target, draft if form == "dense" else None, drafted, g.random(drafts), g.random(n), vocab,
          stride=stride)


LISTS = [
    # drafts of each, vocabulary, entries a list has room for, entries kept
    ([3, 0, 5, 1], 5000, 64, 20),
    ([2, 2], 400, 1, 1),
    ([1] * 20, 151936, 50, 50),
    ([4, 4, 4], 3000, 2500, 2200),    # longer than a chunk of entries
    ([2], 1025, 1025, 1025),
]


@pytest.mark.parametrize("drawn", [True, False])
@pytest.mark.parametrize("case", range(len(LISTS)))
def test_candidate_lists(device, case, drawn):
    lens, vocab, room, keep = LISTS[case]
    g = np.random.default_rng(50 + case)
    drafts, n = sum(lens), len(lens)

    def lists(rows, near=None):
        ids = np.stack([g.permutation(vocab)[:room] for _ in range(rows)]).astype(np.int32)
        p = np.full((rows, room), np.nan, np.float32)
        kept = g.integers(max(1, keep // 2), keep + 1, rows).astype(np.int32)
        for r in range(rows):
            if near is not None:  # most of its tokens are in the other list too
                ids[r, :room] = g.permutation(near[r])
            q = np.sort(probs(g, 1, kept[r], 1.0)[0])[::-1]
            p[r, :kept[r]] = q
        return ids, p, kept

    ids, target, kept = lists(drafts + n)
    row = np.concatenate([np.arange(c) + sum(lens[:s]) + s for s, c in enumerate(lens)]).astype(int)
    q_ids, draft, q_kept = lists(drafts, near=ids[row])
    drafted = np.array([q_ids[r, g.choice(q_kept[r], p=draft[r, :q_kept[r]] / draft[r, :q_kept[r]].astype(np.float64).sum())]
                        for r in range(drafts)], np.int64)
    print("lists", LISTS[case], drawn, flush=True)
    check(device, lens, target, draft if drawn else None, drafted, g.random(drafts), g.random(n), vocab, ids, kept,
          q_ids if drawn else None, q_kept if drawn else None)


def test_rows_and_uniforms_at_their_ends(device):
    nan, inf = float("nan"), float("inf")
    vocab = 9
    base = np.array([0.0, 0.25, nan, 0.5, -1.0, inf, 0.25, 0.0, 0.0], np.float32)
    empty = np.array([0, nan, -inf, inf, 0, 0, -0.0, 0, -2], np.float32)
    # One draft each. target row, draft row, drafted token, uniform, draw
    cases = [
        (base, base, 3, 0.999999, 0.5),        # p = q: accepted
        (base, base, 1, 0.0, 0.0), (base, base, 6, 0.5, 0.999999),
        (base, base, 0, 0.0, 0.3),             # p = 0: never, and p - q is nowhere above zero: drawn from p
        (base, empty, 0, 0.0, 0.3), (empty, base, 3, 0.0, 0.5),  # nothing to draw: -1
        (base, base, 2, 0.1, 0.25), (base, base, 5, 0.1, 0.75),  # NaN and infinity are no probabilities
        (base, empty, 3, 0.9, 1.0),            # q = 0: accepted
        (base, base[::-1].copy(), 8, 0.5, 1.0), (base, base[::-1].copy(), 8, 0.5, nan), (base, base[::-1].copy(), 8, 0.5, -3.0),
        (base, base, -1, 0.0, 0.6), (base, base, 9, 0.0, 0.6), (base, base, 2 ** 31 - 1, 0.0, 0.1),  # no tokens
        (base, base, 3, nan, 0.6), (base, base, 3, 1.0, 0.6),
    ]
    n = len(cases)
    target = np.concatenate([[c[0], base] for c in cases]).astype(np.float32)
    draft = np.stack([c[1] for c in cases])
    drafted, uniforms, draws = (np.array([c[i] for c in cases]) for i in (2, 3, 4))
    lens = [1] * n
    for q in (draft, None):
        accepted, tokens = check(device, lens, target, q, drafted, uniforms, draws, vocab)
        assert tokens[::2][5] == -1
    # The same as lists: every token an entry, in an order of its own.
    g = np.random.default_rng(4)
    order = np.stack([g.permutation(vocab) for _ in range(2 * n)]).astype(np.int32)
    other = np.stack([g.permutation(vocab) for _ in range(n)]).astype(np.int32)
    all_of = lambda m: np.full(m, vocab + 5, np.int32)  # noqa: E731  (more than there is room for)
    for q in (np.take_along_axis(draft, other, 1), None):
        check(device, lens, np.take_along_axis(target, order, 1), q, drafted, uniforms, draws, vocab, order, all_of(2 * n),
              None if q is None else other, None if q is None else all_of(n))


@pytest.mark.parametrize("vocab", [700, 9000, 400000])
def test_draws_of_one_or_more_take_the_last(device, vocab):
    # The last probability is far below the sum's last bit, so running sums in any order may pass the total before it.
    g = np.random.default_rng(vocab)
    n = 12
    target = probs(g, n, vocab, 1.0)
    target[:, -3] = 1e-30
    target[:, -2:] = 0.0
    draws = np.array([1.0, float("nan"), 2.0, float("inf")] * 3, np.float32)
    none = np.zeros(0)
    _, tokens = check(device, [0] * n, target, None, none, none, draws, vocab)
    assert tokens == [vocab - 3] * n
    ids = np.tile(np.arange(vocab, dtype=np.int32), (n, 1))
    _, tokens = check(device, [0] * n, target, None, none, none, draws, vocab, ids, np.full(n, vocab, np.int32))
    assert tokens == [vocab - 3] * n


def test_accepted_borders_are_exact(device):
    # u q against p where they are one unit apart or equal: products of f32 values are exact in f64.
    g = np.random.default_rng(9)
    n, vocab = 256, 64
    target, draft = probs(g, 2 * n, vocab, 1.0), probs(g, n, vocab, 1.0)
    drafted = g.integers(0, vocab, n)
    p, q = target[::2][np.arange(n), drafted].astype(np.float64), draft[np.arange(n), drafted].astype(np.float64)
    u = (p / q).astype(np.float32)
    u[::3] = np.nextafter(u[::3], np.float32(0))
    u[1::3] = np.nextafter(u[1::3], np.float32(9))
    accepted, _ = check(device, [1] * n, target, draft, drafted, u, g.random(n), vocab)
    assert 0 < sum(accepted) < n


def test_captured_calls_and_another_stream(device):
    g = np.random.default_rng(12)
    lens, vocab = [3, 0, 4, 2], 30000
    drafts, n = sum(lens), len(lens)
    h = D.DeviceDrafts(n, vocab)
    target, draft = (dev(probs(g, r, vocab, 2.0), device) for r in (drafts + n, drafts))
    drafted = draft.argmax(1).to(torch.int32)
    starts = dev(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), device)
    u, w = torch.rand(drafts, device=device), torch.rand(n, device=device)
    accepted, tokens = torch.zeros(n, dtype=torch.int32, device=device), torch.zeros(drafts + n, dtype=torch.int32, device=device)
    call = lambda **kw: h.verify(target, drafted, starts, u, w, accepted, tokens, draft=draft, **kw)  # noqa: E731
    call()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        u.copy_(torch.rand(drafts, device=device))
        w.copy_(torch.rand(n, device=device))
        torch.cuda.synchronize()
        call(stream=other.cuda_stream)
        other.synchronize()
        want, want_accepted = tokens.clone(), accepted.clone()
        tokens.fill_(5)
        accepted.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, want) and torch.equal(accepted, want_accepted)


def test_refusals(device):
    h = D.DeviceDrafts(2, 100)
    p, q = torch.zeros(5, 100, device=device), torch.zeros(3, 100, device=device)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731
    u, w, accepted, tokens = torch.zeros(3, device=device), torch.zeros(2, device=device), i32(0, 0), i32(*[0] * 5)
    ids, kept = torch.zeros(5, 100, dtype=torch.int32, device=device), i32(*[1] * 5)

    def refused(code, f, *a, **kw):
        with pytest.raises(R.SamplerError) as e:
            f(*a, **kw)
        assert e.value.code == code

    refused(R.RL_ERR_CAPACITY, h.verify, torch.zeros(6, 100, device=device), i32(0, 0, 0), i32(0, 1, 2, 3), u,
            torch.zeros(3, device=device), i32(0, 0, 0), i32(*[0] * 6))
    refused(R.RL_ERR_ARGUMENT, h.verify, p, i32(0, 0, 0), i32(0, 1, 3), u, w, accepted, tokens, draft=q, target_ids=ids,
            target_kept=kept)  # lists against rows
    refused(R.RL_ERR_ARGUMENT, h.verify, p[:3], i32(0, 0, 0), i32(0), u, w[:0], accepted, i32(0, 0, 0))  # no sequence
    none = i32()
    h.verify(p[:0], none, i32(0), u[:0], w[:0], accepted[:0], tokens[:0])  # nothing to do
