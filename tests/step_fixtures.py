"""Plain statements in float64, on the CPU, of what a drafted serving step adds to the
mixers of mixer_fixtures.py: the short convolution and the state space scan of
include/rl_mixers.h, with bounds of their f32 errors, and the verification of
include/rl_drafts.h. Written from the formulas alone."""
import numpy as np

E = 2.0 ** -24  # half a unit of f32


def silu(y):
    with np.errstate(over="ignore"):
        return y / (1 + np.exp(-y))


def silu_error(y, off):
    """Of silu in f32 of a value that is `off` off: its slope is at most 1.1; the exponent's rounding |y|, the
    exponential, the sum, the reciprocal and the product 8 units together."""
    return 1.1 * off + np.abs(silu(y)) * (np.abs(y) + 8) * E


def conv(x, before, weight, bias, act):
    """x [rows][channels] after the rows `before` [width - 1][channels]. Returns the
    outputs, the state after, and a bound of an f32 evaluation's error."""
    w = weight.shape[1]
    rows = np.concatenate([before, x])
    y, size = np.tile(bias, (len(x), 1)), np.tile(np.abs(bias), (len(x), 1))
    for j in range(w):
        y = y + weight[:, j] * rows[j:j + len(x)]
        size = size + np.abs(weight[:, j] * rows[j:j + len(x)])
    off = size * w * E  # w products added, each rounded once
    if act == "silu":
        y, off = silu(y), silu_error(y, off)
    return y, rows[len(rows) - (w - 1):], off


def scan(x, dt, b, c, z, a, skip, bias, state, softplus=True, pieces=False):
    """One sequence: x, dt, z [rows][channels], b, c [rows][groups][n], state
    [channels][n]. Returns outputs, the state after and bounds of both's f32 errors."""
    h, share = state.copy(), x.shape[1] // b.shape[1]
    size, err = np.abs(h), np.zeros_like(h)
    out, off = np.zeros_like(x), np.zeros_like(x)
    # In pieces a state passes a piece of at most n tokens by the exponential of the sum of its steps: n roundings more of
    # an exponent, of which at most 256 tokens' stand before the last.
    more = 256 if pieces else 0
    for t in range(x.shape[0]):
        v = dt[t] + bias
        s = np.logaddexp(0, v) if softplus else v
        # The step: the sum, an exponential, a logarithm and their corrections, 10 units of the step; of a sum near
        # zero the sum's own rounding counts.
        ds = np.abs(s) * 10 * E + np.abs(v) * E
        e = np.exp(s[:, None] * a)
        bt, ct = np.repeat(b[t], share, 0), np.repeat(c[t], share, 0)
        drive = (s * x[t])[:, None] * bt
        h = e * h + drive
        # The decay: its exponent a s, a rounded to base 2 (2 units with the product), and the exponential 2.
        de = e * (np.abs(a) * (ds[:, None] + np.abs(s)[:, None] * (2 + more) * E) + 4 * E)
        err = e * err + de * size + np.abs(drive) * 4 * E + (ds * np.abs(x[t]))[:, None] * np.abs(bt)
        size = e * size + np.abs(drive)
        err = err + size * E
        y = (h * ct).sum(-1) + skip * x[t]
        o = (err * np.abs(ct)).sum(-1) + ((size * np.abs(ct)).sum(-1) + np.abs(skip * x[t])) * (a.shape[1] + 2) * E
        if z is not None:
            g = silu(z[t])
            o = o * np.abs(g) + np.abs(y) * silu_error(z[t], 0) + np.abs(y * g) * E
            y = y * g
        out[t], off[t] = y, o
    return out, h, off, err


def softened(row):
    """A row's probabilities as they count: no negative, no infinite, no NaN."""
    row = np.asarray(row, np.float64)
    return np.where((row > 0) & np.isfinite(row), row, 0.0)


def verify(target, draft, drafted, uniforms, draw):
    """One sequence. target: len(drafted) + 1 rows, each (ids, probabilities); draft the
    same for each draft, or None. Returns accepted and its tokens."""
    def of(row, token):
        ids, p = row
        return float(softened(p)[np.asarray(ids) == token].sum())

    tokens = []
    for i in range(len(drafted) + 1):
        ids, p = target[i]
        left = p = softened(p)
        if i < len(drafted):
            d = drafted[i]
            q = of(draft[i], d) if draft is not None else 1.0
            if float(np.float64(uniforms[i])) * q < of(target[i], d):
                tokens.append(int(d))
                continue
            if draft is None:
                less = (np.asarray(ids) == d).astype(np.float64)
            else:
                held = dict(zip(np.asarray(draft[i][0]).tolist(), softened(draft[i][1]).tolist()))
                less = np.array([held.get(int(v), 0.0) for v in ids])
            left = np.maximum(p - less, 0.0)
        if not (left > 0).any():
            left = p
        run, at = np.cumsum(left), -1
        if len(run) and run[-1] > 0:
            past = np.flatnonzero((run > max(float(draw) * run[-1], 0.0)) & (left > 0)) if draw == draw else []
            at = int(past[0]) if len(past) else int(np.flatnonzero(left > 0)[-1])
        tokens.append(int(ids[at]) if at >= 0 else -1)
        break
    return len(tokens) - 1, tokens + [-1] * (len(drafted) + 1 - len(tokens))
