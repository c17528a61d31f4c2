"""One set of checks of the 4-bit cache for two places to run it: the GPU, and the CPU execution model of the kernels (tests/emu)."""
import numpy as np
import torch

import cache_reference as ref

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


class World:
    """Where tensors live and the binding that works on them."""

    def __init__(self, cache, device, sync, empty):
        self.cache, self.device, self.sync, self._empty = cache, device, sync, empty

    def put(self, a, dtype=None):
        t = torch.from_numpy(np.ascontiguousarray(a)) if isinstance(a, np.ndarray) else a.contiguous()
        t = t if dtype is None else t.to(dtype)
        out = self._empty(tuple(t.shape), t.dtype)
        out.copy_(t)
        return out

    def full(self, shape, value, dtype):
        return self.put(torch.full(shape, value, dtype=dtype))

    def get(self, t):
        self.sync()
        t = t.detach().cpu()
        return t.double().numpy() if t.dtype.is_floating_point else t.numpy().copy()


class Batch:
    """Sequences of a cache: pages in random order, some left over, tables with entries nobody reads."""

    def __init__(self, world, lengths, rows, heads, d, page, seed=0, bad_pages=(), padding=0, spare_pages=2):
        self.w, self.lengths, self.rows, self.heads, self.d, self.page = world, list(lengths), list(rows), heads, d, page
        self.rng = np.random.default_rng(seed)
        per = [-(-max(0, n) // page) for n in lengths]
        width = max([1] + per)
        self.n_pages = sum(per) + spare_pages
        order = self.rng.permutation(self.n_pages)
        self.table = np.full((len(lengths), width), -7, np.int32)
        at = 0
        for s, n in enumerate(per):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.free = [int(p) for p in order[at:]]
        for s, i, p in bad_pages:
            self.table[s, i] = p
        self.starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.total = int(self.starts[-1]) + padding
        bytes_ = world.cache.page_bytes(heads, d, page)
        # what lies in a page before it is stored to does not matter: ones everywhere are NaNs wherever a number is read
        self.pages = world.full((self.n_pages, bytes_), 255, torch.uint8)
        self.c = world.cache.Cache(self.pages, heads, d, page)
        self.d_table = world.put(self.table)
        self.d_lengths = world.put(np.array(self.lengths, np.int32))
        self.d_starts = world.put(self.starts)

    def fill(self, scale=1.0, edit=None):
        """Stores random rows in all slots of all sequences; edit(k, v, slot of each row) may change them before."""
        total = sum(max(0, n) for n in self.lengths)
        k = (self.rng.standard_normal((total, self.heads, self.d)) * scale + self.rng.standard_normal((1, self.heads, self.d)) * 2).astype(np.float32)
        v = (self.rng.standard_normal((total, self.heads, self.d)) * scale).astype(np.float32)
        if edit:
            edit(k, v, np.concatenate([np.arange(max(0, n)) for n in self.lengths]))
        starts = self.w.put(np.concatenate([[0], np.cumsum([max(0, n) for n in self.lengths])]).astype(np.int32))
        self.c.store(self.w.put(k), self.w.put(v), self.d_table, self.d_lengths, starts)

    def raw(self):
        return ref.Pages(self.w.get(self.pages), self.heads, self.d, self.page)

    def held(self):
        raw = self.raw()
        return [[raw.rows(self.table[s], h, max(0, n)) for h in range(self.heads)] for s, n in enumerate(self.lengths)]


def check_store(world, lengths, rows, heads, d, page, type_, seed=0, make=None, padding=0, strided=False, bad_pages=()):
    """Rows stored are held as the definition says, bit for bit, load as the numbers they stand for, and nothing else changes."""
    b = Batch(world, lengths, rows, heads, d, page, seed, padding=padding, bad_pages=bad_pages)
    before = world.get(b.pages).reshape(-1)
    make = make or (lambda rng, shape: rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[:-1] + (1,))) + rng.standard_normal(shape[1:]))
    kv = [torch.from_numpy(make(b.rng, (b.total, heads, d)).astype(np.float32)).to(TYPES[type_]) for _ in range(2)]
    if strided:   # rows and heads further apart, and off the 16 bytes
        big = [world.full((b.total, heads + 1, d + 3), 9.0, TYPES[type_]) for _ in range(2)]
        for t, x in zip(big, kv):
            t[:, :heads, 1:d + 1] = x.to(t.device)
        dev = [t[:, :heads, 1:d + 1] for t in big]
    else:
        dev = [world.put(x) for x in kv]
    b.c.store(*dev, b.d_table, b.d_lengths, b.d_starts)
    after = world.get(b.pages).reshape(-1)
    raw = b.raw()
    touched = np.zeros(after.shape, bool).reshape(b.n_pages, heads, page // 32, -1)
    expect = [np.zeros((b.total, heads, d)) for _ in range(2)]
    known = np.zeros(b.total, bool)
    for s, n in enumerate(b.lengths):
        for i in range(b.rows[s]):
            slot, r = n - b.rows[s] + i, b.starts[s] + i
            if slot < 0:
                continue
            known[r] = True
            p = int(b.table[s, slot // page])
            if not 0 <= p < b.n_pages:
                continue
            for h in range(heads):
                got_k, got_v, places = raw.row(p, h, slot % page)
                touched[p, h, slot % page // 32, places] = True
                for x, got, out in ((kv[0], got_k, expect[0]), (kv[1], got_v, expect[1])):
                    x = x[r, h].double().numpy()
                    want = ref.quantise(x)
                    for a, w, what in zip(got, want, ("codes", "s", "lo")):
                        assert np.array_equal(np.asarray(a, np.float64), np.asarray(w, np.float64), equal_nan=True), (what, s, i, h, a, w)
                    out[r, h] = ref.values(*want)
                    off = np.abs(out[r, h] - x) - np.repeat(want[1], 32) / 2
                    assert not (off > 1e-12 * np.abs(x)).any(), "the error bound s / 2"
    assert np.array_equal(after[~touched.reshape(-1)], before[~touched.reshape(-1)]), "bytes of other slots changed"
    # back as numbers, into arrays whose other rows stay as they are
    wide = [world.full((b.total, heads + 1, d + 3), 77.0, TYPES[type_]) for _ in range(2)]
    outs = [x[:, :heads, 1:d + 1] for x in wide] if strided else [world.full((b.total, heads, d), 77.0, TYPES[type_]) for _ in range(2)]
    b.c.load(*outs, b.d_table, b.d_lengths, b.d_starts)
    for x in wide if strided else []:
        x = world.get(x)
        assert (x[:, heads:] == 77.0).all() and (x[:, :, 0] == 77.0).all() and (x[:, :, d + 1:] == 77.0).all(), "what lies between rows was written"
    for out, want in zip(outs, expect):
        got = world.get(out)
        assert (got[~known] == 77.0).all(), "padding was written"
        # lo + s c is one rounding to 32 bits, the type another
        tol = (ref.EPS[type_] + 2.0 ** -24) * np.abs(want) + (6e-8 if type_ == "f16" else 0.0)
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got[known]), nan[known])
        over = np.abs(want) >= 65504 if type_ == "f16" else np.zeros(want.shape, bool)
        assert ((np.abs(got - want) <= tol) | nan | over)[known].all()
    return b


def check_attend(world, lengths, rows, heads, group, d, page, type_, causal=True, window=0, scale=None, weights=False, in_place=False, seed=0,
                 padding=0, bad_pages=(), strided=False, q_scale=1.0, tight=True, q_edit=None, fill_scale=1.0, prior=True, edit=None):
    b = Batch(world, lengths, rows, heads, d, page, seed, padding=padding, bad_pages=bad_pages)
    b.fill(fill_scale, edit)
    q = torch.from_numpy((b.rng.standard_normal((b.total, heads * group, d)) * q_scale).astype(np.float32)).to(TYPES[type_])
    if q_edit:
        q_edit(q)
    if strided:
        big = world.full((heads * group, b.total, d + 5), 3.0, TYPES[type_])
        big[:, :, 3:d + 3] = q.transpose(0, 1).to(big.device)
        dq = big[:, :, 3:d + 3].transpose(0, 1)
        big_out = world.full((b.total, d // 2 + heads * group * d), 55.0, TYPES[type_])
        out = big_out.as_strided((b.total, heads * group, d), (big_out.stride(0), d, 1), d // 2)
    else:
        dq, out = world.put(q), world.full((b.total, heads * group, d), 55.0, TYPES[type_])
    lse = world.full((b.total, heads * group), 44.0, torch.float32)
    held = b.held()
    most = max([1] + [n for n in lengths])
    width = most + 3 if tight else b.table.shape[1] * page   # (what the default of max_length asks for)
    first = np.abs(b.rng.standard_normal((len(lengths), heads, width))).astype(np.float32)
    kw = {}
    if weights:
        kw["weights"] = world.put(first) if in_place else world.full(first.shape, 33.0, torch.float32)
        if prior:
            kw["prior"] = kw["weights"] if in_place else world.put(first)
    if tight:
        kw.update(max_rows=max([0] + list(rows)), max_length=most)
    need = b.c.scratch_bytes(b.total, heads * group, len(lengths), b.table.shape[1], TYPES[type_], window=window, weights=weights, lse=True,
                             max_rows=kw.get("max_rows"), max_length=kw.get("max_length"))
    kw["scratch"] = world.full((need // 4 + 4,), float("nan"), torch.float32)
    b.c.attend(dq, out, b.d_table, b.d_lengths, b.d_starts, scale=scale, causal=causal, window=window, lse=lse, **kw)
    sc = d ** -0.5 if scale is None else scale
    keys, vals, there = ([[x[i] for x in per] for per in held] for i in range(3))
    want, want_lse, want_w, tol, tol_lse, tol_w = ref.attention(q.double().numpy(), keys, vals, there, [max(0, n) for n in lengths], b.starts, group,
                                                               float(np.float32(sc)), causal, window, type_, first if weights and prior else None)
    got, got_lse = world.get(out), world.get(lse)
    n = int(b.starts[-1])
    assert (got[n:] == 55.0).all() and (got_lse[n:] == 44.0).all(), "padding was written"
    empty = np.isneginf(want_lse[:n])
    assert np.array_equal(np.isneginf(got_lse[:n]), empty)
    assert (got[:n][empty] == 0).all()
    close(got_lse[:n][~empty], want_lse[:n][~empty], tol_lse[:n][~empty], "lse")
    close(got[:n], want[:n], tol[:n], "out")
    if weights:
        got_w = world.get(kw["weights"])
        for s, L in enumerate(lengths):
            L = max(0, L)
            close(got_w[s, :, :L], want_w[s], tol_w[s], "weights")
            assert (got_w[s, :, L:] == (first[s, :, L:] if in_place else 33.0)).all(), "weights behind the last slot"
    if strided:
        rest = world.get(big_out)
        assert (rest[:, :d // 2] == 55.0).all()
    return got[:n], got_lse[:n]


def close(got, want, tol, what):
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaNs at other places"
    fine = ~np.isnan(want)
    off = np.abs(got[fine] - want[fine])
    bad = ~(off <= tol[fine])
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(off / np.maximum(tol[fine], 1e-300))} times what is allowed"


def check_evict(world, lengths, heads, d, page, keep, first=0, recent=0, seed=0, make=None, bad_pages=()):
    b = Batch(world, lengths, [1] * len(lengths), heads, d, page, seed, bad_pages=bad_pages, spare_pages=2 + len(lengths) * -(-keep // page))
    b.fill()
    most = max([1] + list(lengths))
    w = (make or (lambda rng, shape: rng.random(shape) ** 4))(b.rng, (len(lengths), heads, most + 5)).astype(np.float32)
    width = -(-keep // page)
    to_table = np.array([[b.free.pop() for _ in range(width)] for _ in lengths], np.int32).reshape(len(lengths), width)
    to_lengths = world.full((len(lengths),), 99, torch.int32)
    before = b.raw()
    old = world.get(b.pages)
    to_weights, kept = b.c.evict(world.put(w), b.d_table, b.d_lengths, keep, world.put(to_table), to_lengths, first=first, recent=recent, max_length=most,
                                 to_weights=world.full((len(lengths), heads, keep), 5.0, torch.float32),
                                 kept=world.full((len(lengths), heads, keep), 5, torch.int32))
    got_w, got_kept = world.get(to_weights), world.get(kept)
    assert world.get(to_lengths).tolist() == [min(max(0, n), keep) for n in lengths]
    stays = ref.evict(w, [max(0, n) for n in lengths], keep, first, recent)
    after = b.raw()
    for s, n in enumerate(lengths):
        for h in range(heads):
            want = stays[s * heads + h]
            assert got_kept[s, h, :len(want)].tolist() == want
            assert (got_kept[s, h, len(want):] == -1).all() and (got_w[s, h, len(want):] == 0).all()
            assert np.array_equal(got_w[s, h, :len(want)], w[s, h][want].astype(np.float64), equal_nan=True)
            for i, slot in enumerate(want):
                p = int(b.table[s, slot // page])
                new = after.row(int(to_table[s, i // page]), h, i % page)
                if 0 <= p < b.n_pages:
                    was = before.row(p, h, slot % page)
                    for x, y in zip(new[0] + new[1], was[0] + was[1]):
                        assert np.array_equal(x, y, equal_nan=True)
                else:
                    assert not ref.values(*new[0]).any() and not ref.values(*new[1]).any()
    used = set(to_table.reshape(-1).tolist())
    now = world.get(b.pages)
    for p in range(b.n_pages):
        assert p in used or np.array_equal(now[p], old[p]), "a page that was not named changed"
    return b


# Rows of keys and values that do not fit float16 numbers, or are none: what kernels take another way for.
def huge_values(k, v, slots):
    v[slots // 32 % 3 == 1] *= 9e3


def tiny_values(k, v, slots):
    v[slots // 32 % 2 == 0] *= 1e-6
    v[slots % 32 == 7] = 1e-9      # a block of one small number: s = 0


def tiny_keys(k, v, slots):
    k[slots // 32 % 2 == 1] *= 1e-6


def late_nan(k, v, slots):
    """Only the last two rows of a causal batch see it."""
    v[slots >= slots.max() - 1, 0, 3] = np.nan


def late_nan_key(k, v, slots):
    k[slots >= slots.max() - 1, 0, 3] = np.inf


def check_run(world, heads=2, group=3, d=64, page=32, type_="bf16", seed=3, first=(37, 5, 50), steps=3, keep=24):
    """As a server would: prompts stored and attended with their weights counted, tokens one by one, eviction to other pages, more tokens."""
    rng = np.random.default_rng(seed)
    n, t = len(first), TYPES[type_]
    width = -(-(max(first) + 2 * steps) // page)
    order = rng.permutation(2 * n * width + 1)
    table = order[:n * width].reshape(n, width).astype(np.int32)
    other = order[n * width:2 * n * width].reshape(n, width).astype(np.int32)
    pages = world.full((len(order), world.cache.page_bytes(heads, d, page)), 255, torch.uint8)
    c = world.cache.Cache(pages, heads, d, page)
    most = width * page
    d_table, d_other = world.put(table), world.put(other)
    weights = world.full((n, heads, most), 0.0, torch.float32)
    book = np.zeros((n, heads, most))
    slack = np.zeros((n, heads, most))
    lengths = np.zeros(n, np.int32)

    def step(rows):
        nonlocal lengths
        lengths = (lengths + rows).astype(np.int32)
        starts = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        k, v = (torch.from_numpy(rng.standard_normal((starts[-1], heads, d)).astype(np.float32)).to(t) for _ in range(2))
        q = torch.from_numpy(rng.standard_normal((starts[-1], heads * group, d)).astype(np.float32)).to(t)
        d_lengths, d_starts = world.put(lengths), world.put(starts)
        c.store(world.put(k), world.put(v), d_table, d_lengths, d_starts)
        out = world.full(tuple(q.shape), 0.0, t)
        need = c.scratch_bytes(len(q), heads * group, n, width, t, weights=True)
        c.attend(world.put(q), out, d_table, d_lengths, d_starts, weights=weights, prior=weights, scratch=world.full((need // 4 + 4,), float("nan"), torch.float32))
        raw = ref.Pages(world.get(pages), heads, d, page)
        held = [[raw.rows(now[s], h, int(L)) for h in range(heads)] for s, L in enumerate(lengths)]
        part = [[[x[i] for x in per] for per in held] for i in range(3)]
        want, _, w, tol, _, tol_w = ref.attention(q.double().numpy(), *part, lengths, starts, group, d ** -0.5, True, 0, type_, book)
        close(world.get(out), want, tol, "out")
        got = world.get(weights)
        for s, L in enumerate(lengths):
            slack[s, :, :L] += tol_w[s]
            close(got[s, :, :L], w[s], slack[s, :, :L], "weights")
            book[s, :, :L] = w[s]

    now = table
    step(np.array(first))
    for _ in range(steps):
        step(np.ones(n, np.int32))
    to_lengths = world.full((n,), 0, torch.int32)
    old = world.get(weights)
    to_weights, kept = c.evict(weights, d_table, world.put(lengths), keep, d_other, to_lengths, first=2, recent=8,
                               to_weights=world.full((n, heads, keep), 0.0, torch.float32), kept=world.full((n, heads, keep), 0, torch.int32))
    stays = ref.evict(old, lengths, keep, 2, 8)
    got, got_w = world.get(kept), world.get(to_weights)
    book[:], slack[:] = 0.0, 0.0
    for s, L in enumerate(lengths):
        for h in range(heads):
            row = stays[s * heads + h]
            assert got[s, h, :len(row)].tolist() == row
            book[s, h, :len(row)] = old[s, h][row]
    lengths = world.get(to_lengths).astype(np.int32)
    assert lengths.tolist() == [min(keep, n + steps) for n in first]
    now, d_table = other, d_other
    weights = world.put(book, torch.float32)
    for _ in range(steps):
        step(np.resize([1, 0, 2], n))
