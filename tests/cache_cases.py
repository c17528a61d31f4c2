"""Further checks of the 4-bit cache for both places to run it (cache_world.py): calls in which not all is as wide as it could be."""
from fractions import Fraction

import numpy as np
import torch

import cache_reference as ref
from cache_world import TYPES, Batch, close


def weights_of_rows(q, k, there, rows, n, L, group, scale, causal, window):
    """The attention that one head's slots receive from rows `rows` (of n) of a sequence of L slots, and how far it may be off: a weight is off
    by a factor of 1 + 2 e + run + |lse| 2^-22 as cache_reference.attention derives them, the running sum by a rounding for each row."""
    d = q.shape[-1]
    w, dw, j = np.zeros(L), np.zeros(L), np.arange(L)
    for i in rows:
        at = L - n + i
        see = there & ((j <= at) if causal else True) & ((j > at - window) if window else True)
        if not see.any():
            continue
        for g in range(group):
            s = scale * (k[see] @ q[i, g])
            size = abs(scale) * (np.abs(k[see]) + 2 * np.abs(k[see]).max(-1, keepdims=True)) @ np.abs(q[i, g])
            z = s.max() + np.log(np.exp(s - s.max()).sum())
            p = np.exp(s - z)
            e, run = (64 + d / 32) * 2.0 ** -24 * size.max(), 2.0 ** -20 + L * 2.0 ** -24
            w[see] += p
            dw[see] += p * (2 * e + run + abs(z) * 2.0 ** -22) + 2.0 ** -23 * w[see]
    return w, dw


def check_rows_left_out(world, lengths, rows, heads, group, d, page, type_, causal, window, max_rows=None, hold=None, seed=0):
    """Sequences with more rows than max_rows, or than the arrays hold: the rows that stay get what they get when nothing is left out, the others
    are left as they were, and weights count the rows that stay."""
    b = Batch(world, lengths, rows, heads, d, page, seed)
    b.fill()
    hold = b.total if hold is None else hold
    q = torch.from_numpy(b.rng.standard_normal((b.total, heads * group, d)).astype(np.float32)).to(TYPES[type_])
    out, lse = world.full((hold, heads * group, d), 55.0, TYPES[type_]), world.full((hold, heads * group), 44.0, torch.float32)
    width = b.table.shape[1] * page
    weights = world.full((len(lengths), heads, width), 33.0, torch.float32)
    need = b.c.scratch_bytes(hold, heads * group, len(lengths), b.table.shape[1], TYPES[type_], window=window, weights=True, lse=True, max_rows=max_rows)
    b.c.attend(world.put(q[:hold]), out, b.d_table, b.d_lengths, b.d_starts, causal=causal, window=window, max_rows=max_rows, lse=lse, weights=weights,
               scratch=world.full((need // 4 + 4,), float("nan"), torch.float32))
    held = b.held()
    keys, vals, there = ([[x[i] for x in per] for per in held] for i in range(3))
    scale, q = float(np.float32(d ** -0.5)), q.double().numpy()
    want, want_lse, _, tol, tol_lse, _ = ref.attention(q, keys, vals, there, lengths, b.starts, group, scale, causal, window, type_)
    got, got_lse, got_w = world.get(out), world.get(lse), world.get(weights)
    most = hold if max_rows is None else max_rows
    for s, (L, n) in enumerate(zip(lengths, rows)):
        first = int(b.starts[s])
        stay = [i for i in range(n) if i < most and first + i < hold]
        gone = [first + i for i in range(n) if i not in stay and first + i < hold]
        at = [first + i for i in stay]
        close(got_lse[at], want_lse[at], tol_lse[at], f"lse of sequence {s}")
        close(got[at], want[at], tol[at], f"out of sequence {s}")
        assert (got[gone] == 55.0).all() and (got_lse[gone] == 44.0).all(), "rows that are left out were written"
        for h in range(heads):
            part = q[first:first + n, h * group:(h + 1) * group]
            w, dw = weights_of_rows(part, keys[s][h], there[s][h], stay, n, L, group, scale, causal, window)
            close(got_w[s, h, :L], w, dw + 2.0 ** -24 * w, f"weights of sequence {s}")
        assert (got_w[s, :, L:] == 33.0).all()


# Constant blocks far from the others: held exactly (s = 0) up to bfloat16's largest number.
LARGEST = float(torch.tensor(0x7f7f, dtype=torch.int16).view(torch.bfloat16))


def far_values(k, v, slots):
    v[slots % 5 == 2] = 2.0 ** 66


def farthest_values(k, v, slots):
    v[slots % 7 == 3] = float(torch.tensor(1e38).bfloat16())
    v[slots % 32 == 9] = -LARGEST


def only_farthest_values(k, v, slots):
    v[:] = LARGEST


def last_value_far(k, v, slots):
    """Seen by the last row of a causal batch alone, or the last columns."""
    v[slots == slots.max()] = LARGEST


def far_and_tiny_values(k, v, slots):
    v[slots % 11 == 4] = 2.0 ** 41
    v[slots % 3 == 0] = 2.0 ** -40


FAR = [far_values, farthest_values, only_farthest_values, last_value_far, far_and_tiny_values]


# ---------------------------------------------------------------- the codec's decisions in exact arithmetic
POSITIVE = [Fraction(float(v)) for v in ref.bf16_values(np.arange(0x7f80))]                             # 0 and the positive bfloat16, ascending
STEPS = [Fraction(float(v)) for v in np.arange(0x7c00, dtype=np.uint16).view(np.float16)]


def exact_block(x):
    """(codes, s, lo) of 32 finite numbers of 32 bits from the header's definition, in rational numbers."""
    x = [Fraction(float(v)) for v in x]
    low, high = min(x), max(x)
    up, steps = POSITIVE, STEPS
    if low >= 0:
        a, b = 0, len(up) - 1                                  # the largest not above
        while a < b:
            m = (a + b + 1) // 2
            a, b = (m, b) if up[m] <= low else (a, m - 1)
        lo = up[a]
    else:
        a, b = 0, len(up) - 1                                  # of the negated ones the smallest not below
        while a < b:
            m = (a + b) // 2
            a, b = (a, m) if up[m] >= -low else (m + 1, b)
        lo = -up[a]
    if 15 * steps[-1] < high - lo:
        return [0] * 32, float("nan"), 0.0
    a, b = 0, len(steps) - 1
    while a < b:
        m = (a + b) // 2
        a, b = (a, m) if 15 * steps[m] >= high - lo else (m + 1, b)
    s = steps[a]
    codes = [0 if s == 0 else sum(v >= lo + (j + Fraction(1, 2)) * s for j in range(15)) for v in x]
    return codes, float(s), float(lo)


def hard_blocks(seed=0, n=40):
    """Blocks whose borders take more than 64 bits: a lowest number far below the step, exact half steps, their neighbours."""
    rng = np.random.default_rng(seed)
    out = [[1e-30, 15, 0.5, 2.5] + [1] * 28, [-1e-30, 15, 0.5, 2.5, 14.5] + [1] * 27, [1e-30, 30, 1, 3, 5, 29] + [2] * 26,
           [-1e-30, 30, 1, 3, 5, 29] + [2] * 26, [-0.5, 14.5, 1e-30, -1e-30, 0.0, -0.0, 1e-45, -1e-45] + [3] * 24,
           [1e-45, 2.0 ** -24 * 15, 2.0 ** -25, 3 * 2.0 ** -25] + [0.0] * 28, [-1e-45, 2.0 ** -24 * 15, 2.0 ** -25, 3 * 2.0 ** -25] + [0.0] * 28,
           [-1e-40] * 31 + [1e-40], [1e-40, 65504.0 * 15] + [32752.0] * 30, [-1e-40, 65504.0 * 15] + [1.0] * 30]
    for _ in range(n):
        s = float(np.float16(2.0 ** rng.integers(-20, 12) * rng.integers(1024, 2048) / 1024))
        lo = float(torch.tensor(rng.choice([-1, 1]) * 2.0 ** float(rng.integers(-120, 12))).bfloat16())
        at = lo + (rng.integers(0, 15, 32) + rng.choice([0.0, 0.5], 32)) * s
        x = at.astype(np.float32)
        x = np.where(rng.random(32) < 0.3, np.nextafter(x, np.float32(np.inf)), np.where(rng.random(32) < 0.3, np.nextafter(x, np.float32(-np.inf)), x))
        x[0], x[1] = lo, np.float32(lo + 15 * s)
        out.append(np.maximum(x, np.float32(lo)).tolist())
    return np.array(out, np.float32)


def check_store_exact(world, blocks):
    """Codes, steps and lowest numbers bit for bit what rational arithmetic says, keys and values."""
    n = len(blocks) // 2
    b = Batch(world, [n], [n], 1, 64, 32)
    x = world.put(np.ascontiguousarray(blocks[:2 * n].reshape(n, 1, 64)))
    b.c.store(x, x, b.d_table, b.d_lengths, b.d_starts)
    raw = b.raw()
    for r in range(n):
        key, value, _ = raw.row(int(b.table[0, r // 32]), 0, r % 32)
        for i in range(2):
            codes, s, lo = exact_block(blocks[2 * r + i])
            for got, what in ((key, "key"), (value, "value")):
                assert np.array_equal([got[1][i], got[2][i]], [s, lo], equal_nan=True), (what, blocks[2 * r + i], got[1][i], s, got[2][i], lo)
                assert got[0][32 * i:32 * i + 32].tolist() == codes, (what, blocks[2 * r + i])


# ---------------------------------------------------------------- scores of 2^26 that lie a few units apart
def close_keys(k, v, slots):
    """Score 6.3e7 + 2.77 c with the queries below, c = 2 more from record to record: exponents of two that rise by about 8."""
    k[:] = 0.0
    k[:, :, 0] = 7680.0
    k[:, :, 32] = (2 * (slots // 32) % 16)[:, None]
    k[:, :, 33] = 15.0


def close_queries(q):
    q[:] = 0.0
    q[:, :, 0] = 8192.0
    q[:, :, 32] = 2.77


# ---------------------------------------------------------------- queries and scales near the end of 32 bits, scores inside it
def small_constant_keys(k, v, slots):
    k[:] = (2.0 ** -100 * (1 + slots % 7 / 8.0))[:, None, None]


def largest_queries(q):
    """Columns of 2^121 and more beside ordinary ones and small ones."""
    q[:, 0] *= 2.0 ** 122
    q[:, 1:2] *= 2.0 ** 60
    q[-1, -1] *= 2.0 ** -20


FAR_QUERIES = [
    dict(q_scale=1e37), dict(q_scale=1e37, scale=1e-3), dict(q_scale=1e5, scale=1e31), dict(q_scale=3.0, scale=-1e36), dict(q_scale=1e37, scale=1e-37),
    dict(q_edit=largest_queries, edit=small_constant_keys), dict(q_edit=largest_queries, scale=0.01), dict(q_scale=1e-30, scale=1e37)]


def check_weights_of_large_scores(world, rows, group, type_, q_scale):
    """Scores far above 2^16, where lse in 32 bits no longer says which share a slot has: a weight is still between 0 and the number of rows and
    heads that count, and what lies outside what they see gets none."""
    b = Batch(world, [90], [rows], 1, 64, 32, seed=2)
    b.fill()
    q = world.put((b.rng.standard_normal((rows, group, 64)) * q_scale).astype(np.float32), TYPES[type_])
    out, weights = world.full((rows, group, 64), 0.0, TYPES[type_]), world.full((1, 1, 96), 33.0, torch.float32)
    need = b.c.scratch_bytes(rows, group, 1, 3, TYPES[type_], weights=True)
    b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, weights=weights, scratch=world.full((need // 4 + 4,), float("nan"), torch.float32))
    w = world.get(weights)[0, 0]
    assert (w[:90] >= 0).all() and (w[:90] <= rows * group * (1 + rows * group * 2.0 ** -24)).all() and (w[90:] == 33.0).all(), w
    assert (w[90 - np.arange(rows)[::-1] - 1] <= (np.arange(rows, 0, -1)) * group * (1 + 2.0 ** -20)).all()
    assert np.isfinite(world.get(out)).all()


def check_lse_without_and_with_weights(world, type_, d, lengths=(300, 40)):
    """The same scores whether or not weights are asked for: out and lse bit for bit."""
    b = Batch(world, lengths, [2] * len(lengths), 2, d, 32, seed=3)
    b.fill()
    q = world.put(b.rng.standard_normal((b.total, 6, d)).astype(np.float32), TYPES[type_])
    results = []
    for weights in (False, True):
        out, lse = world.full((b.total, 6, d), 0.0, TYPES[type_]), world.full((b.total, 6), 0.0, torch.float32)
        width = b.table.shape[1] * 32
        need = b.c.scratch_bytes(b.total, 6, len(lengths), b.table.shape[1], TYPES[type_], weights=weights, lse=True, max_rows=2)
        kw = dict(weights=world.full((len(lengths), 2, width), 0.0, torch.float32)) if weights else {}
        b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, lse=lse, max_rows=2, scratch=world.full((need // 4 + 4,), float("nan"), torch.float32), **kw)
        results.append((world.get(out), world.get(lse)))
    assert np.array_equal(results[0][0], results[1][0]) and np.array_equal(results[0][1], results[1][1])
