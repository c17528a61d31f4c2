"""The 4-bit cache on the GPU, against the definition in 64 bits (tests/cache_reference.py)."""
import cache_reference as ref
import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from cache_world import (TYPES, Batch, World, check_attend, check_evict, check_run, check_store, close, huge_values, late_nan, late_nan_key,
                         tiny_keys, tiny_values)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def world(cuda):
    import importlib
    entry.load_package()
    cache = importlib.import_module(entry.PKG_NAME + ".cache")
    if not isinstance(cuda, type(torch)):
        pytest.skip("runs on the GPU; tests/test_emu_cache.py holds what the CPU model can finish")
    return World(cache, "cuda", torch.cuda.synchronize, lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda"))


from test_emu_cache import blocks  # noqa: E402


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,rows,heads,d,page", [
    ([1], [1], 1, 64, 32),
    ([40, 33, 0, 129], [7, 33, 0, 129], 3, 128, 32),
    ([5, 200], [2, 150], 2, 256, 64),
    ([3, 4], [5, 4], 5, 64, 128),
])
def test_store_and_load(world, lengths, rows, heads, d, page, type_):
    check_store(world, lengths, rows, heads, d, page, type_, padding=3)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
def test_store_hard_blocks(world, type_):
    check_store(world, [130], [130], 2, 128, 64, type_, make=blocks)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_store_strided_and_bad_pages(world, d):
    check_store(world, [40], [40], 2, d, 32, "bf16", strided=True)
    check_store(world, [70, 33], [70, 33], 1, d, 32, "f32", bad_pages=[(0, 1, -1), (1, 0, 1 << 30)], strided=True)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,rows,heads,group,d,page,kw", [
    ([1], [1], 1, 1, 64, 32, {}),
    ([33, 64, 31, 32], [1, 1, 1, 1], 2, 3, 64, 32, {}),
    ([700, 45], [1, 1], 2, 4, 128, 64, {}),
    ([70, 3], [20, 3], 1, 5, 128, 64, dict(padding=3)),
    ([90, 0, 5], [3, 0, 7], 2, 2, 64, 32, {}),
    ([150], [40], 1, 3, 256, 32, {}),
    ([150, 77], [6, 9], 1, 3, 128, 32, dict(causal=False)),
    ([190], [9], 1, 2, 64, 32, dict(window=11)),
    ([190, 50], [30, 50], 2, 2, 128, 32, dict(window=40, weights=True)),
    ([90], [4], 1, 2, 64, 32, dict(window=1, causal=False, scale=0.5)),
    ([64], [3], 2, 2, 128, 32, dict(strided=True)),
    ([196], [3], 1, 2, 64, 64, dict(bad_pages=[(0, 1, -1)], weights=True)),
    ([170, 20], [5, 0], 2, 3, 64, 32, dict(weights=True, in_place=True, tight=False)),
    ([135], [2], 1, 20, 128, 32, dict(weights=True, prior=False)),
    ([300], [1], 1, 1, 128, 64, dict(q_scale=30.0)),                  # nearly all on one slot
    ([300], [17], 1, 16, 64, 64, dict(fill_scale=1e-3, q_scale=1e-2, weights=True)),
])
def test_attend(world, lengths, rows, heads, group, d, page, type_, kw):
    check_attend(world, lengths, rows, heads, group, d, page, type_, **kw)


@pytest.mark.parametrize("lengths,heads,d,page,keep,first,recent", [
    ([50], 1, 64, 32, 20, 2, 5),
    ([1300, 10, 0, 1025], 3, 128, 32, 333, 0, 33),
    ([140], 2, 64, 64, 140, 1, 1),
    ([133], 1, 256, 32, 1, 0, 0),
    ([2500], 1, 64, 128, 1100, 4, 1000),
    ([90, 91], 2, 64, 32, 90, 45, 45),
])
def test_evict(world, lengths, heads, d, page, keep, first, recent):
    check_evict(world, lengths, heads, d, page, keep, first, recent)


def test_evict_ties_and_odd_weights(world):
    def odd(rng, shape):
        w = rng.integers(0, 3, shape).astype(np.float64)
        w[..., ::7] = np.nan
        w[..., 1::11] = -0.0
        w[..., 2::13] = -1.0
        w[..., 3::17] = np.inf
        return w
    check_evict(world, [160, 45], 2, 64, 32, 61, 3, 4, make=odd, bad_pages=[(0, 1, 5000)])


# Many columns: records unpacked once for several tiles of sixteen (16-bit results), and what falls back from there.
@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("lengths,rows,heads,group,d,page,kw", [
    ([100], [33], 1, 2, 64, 32, {}),                                    # 5 tiles
    ([170, 33, 0], [60, 2, 0], 2, 4, 128, 32, dict(padding=1)),         # 15 tiles, of the second sequence one
    ([90], [40], 1, 2, 256, 32, dict(strided=True)),
    ([90], [75], 1, 8, 256, 64, {}),                                    # 38 tiles
    ([700], [9], 1, 2, 64, 32, dict(window=30)),                        # parts
    ([900, 30], [9, 9], 2, 4, 128, 64, dict(weights=True)),
    ([90], [9], 1, 4, 64, 32, dict(causal=False, weights=True)),
    ([230], [10], 1, 3, 128, 32, dict(edit=huge_values)),
    ([130], [10], 1, 3, 64, 32, dict(edit=tiny_values, weights=True)),
    ([130], [10], 1, 3, 256, 32, dict(edit=tiny_keys)),
    ([70], [8], 1, 3, 64, 32, dict(edit=late_nan)),
    ([70], [8], 1, 3, 128, 32, dict(edit=late_nan_key, weights=True)),
    ([200], [10], 1, 3, 64, 32, dict(bad_pages=[(0, 1, 99), (0, 4, -1)])),
    ([20], [33], 1, 2, 64, 32, {}),                                     # more rows than slots
    ([320], [300], 1, 1, 64, 32, dict(window=40)),                      # a tile sees a part of what its parts are cut from
    ([320], [300], 1, 1, 128, 32, dict(window=40, edit=huge_values)),
    ([600, 340], [300, 2], 2, 2, 64, 64, dict(window=260, weights=True, edit=tiny_values)),
])
def test_attend_many_columns(world, lengths, rows, heads, group, d, page, type_, kw):
    check_attend(world, lengths, rows, heads, group, d, page, type_, **kw)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("edit", [huge_values, tiny_values, tiny_keys, late_nan, late_nan_key])
def test_attend_hard_rows(world, edit, d, type_):
    check_attend(world, [300, 64], [3, 1], 1, 2, d, 32, type_, edit=edit)


@pytest.mark.parametrize("group", [1, 16, 17, 256])
def test_attend_groups(world, group):
    check_attend(world, [90], [1], 1, group, 64, 32, "bf16", weights=True)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
def test_operators_together(world, type_):
    check_run(world, type_=type_, d=128)
    check_run(world, type_=type_, group=8, first=(80, 1, 33, 64), keep=31, seed=4)


def decode_setup(world, lengths, heads=2, group=4, d=128, page=32, seed=1, type_="bf16", room=96):
    """A filled cache whose tables have room for more slots, and one new row for each sequence."""
    b = Batch(world, [room] * len(lengths), [1] * len(lengths), heads, d, page, seed)
    b.fill()
    b.lengths = list(lengths)
    b.d_lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    n = len(lengths)
    x = [world.put(b.rng.standard_normal((n, h, d)).astype(np.float32), TYPES[type_]) for h in (heads, heads, heads * group)]
    return b, x, world.full((n, heads * group, d), 0.0, TYPES[type_]), world.full((n, heads, room), 0.0, torch.float32)


def test_same_bits_every_time(world):
    b, (k, v, q), out, w = decode_setup(world, [90, 5, 64])
    b.c.store(k, v, b.d_table, b.d_lengths, b.d_starts)
    results = []
    for _ in range(4):
        b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, weights=w)
        results.append((out.clone(), w.clone()))
    for o, x in results[1:]:
        assert torch.equal(o, results[0][0]) and torch.equal(x, results[0][1])


def test_rows_alone_and_together_agree(world):
    """A sequence's bits do not depend on its neighbours in the batch, as long as it is cut into the same parts."""
    b, (k, v, q), out, _ = decode_setup(world, [90, 5, 64])
    b.c.store(k, v, b.d_table, b.d_lengths, b.d_starts)
    b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts)
    one = torch.zeros_like(out)
    for s in range(3):
        starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        b.c.attend(q[s:s + 1], one[s:s + 1], b.d_table[s:s + 1], b.d_lengths[s:s + 1], starts)
    scale = out.float().abs().max()
    assert ((one.float() - out.float()).abs() <= 2 * ref.EPS["bf16"] * scale).all()


def test_captured_and_replayed(world):
    """Store, attention with its weights counted, and eviction in one graph; new rows, lengths and tables between the replays, and
    the program's own work on the same memory; every replay gives the bits of the same calls made one by one."""
    b, (k, v, q), out, w = decode_setup(world, [90, 5, 64])
    prior = world.put(b.rng.random(tuple(w.shape)).astype(np.float32))
    extra = Batch(world, [32] * 3, [1] * 3, 2, 128, 32)   # (for its tables alone)
    pages = torch.cat([b.pages, extra.pages])
    c = world.cache.Cache(pages, 2, 128, 32)
    to_table = extra.d_table + b.n_pages
    to_lengths = world.full((3,), 0, torch.int32)
    to_w, kept = world.full((3, 2, 24), 0.0, torch.float32), world.full((3, 2, 24), 0, torch.int32)

    def calls():
        c.store(k, v, b.d_table, b.d_lengths, b.d_starts)
        c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, weights=w, prior=prior)
        c.evict(w, b.d_table, b.d_lengths, 24, to_table, to_lengths, first=1, recent=4, to_weights=to_w, kept=kept)

    def results():
        return [x.clone() for x in (pages, out, w, to_lengths, to_w, kept)]

    before = pages.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        calls()
    for step in range(5):
        b.d_lengths.copy_(torch.tensor([[90, 5, 64], [91, 6, 65], [96, 1, 32], [33, 0, 0], [64, 25, 24]][step], dtype=torch.int32))
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, device="cuda") * (1 + step))
        pages.copy_(before)
        calls()
        want = results()
        torch.cuda.synchronize()
        pages.copy_(before)
        for x in (out, w, to_lengths, to_w, kept):
            x.zero_()
        # (what lies behind a sequence's last slot is left as it was: the same start for both)
        want[2] = torch.where(torch.arange(96, device="cuda")[None, None] < b.d_lengths[:, None, None], want[2], torch.zeros_like(want[2]))
        g.replay()
        got = results()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), step


def test_two_graphs_side_by_side(world):
    """Each captured call has scratch memory of its own: replays on two streams at once give what they give alone."""
    sets = [decode_setup(world, [1500, 700], room=1504, seed=i) for i in (1, 2)]
    graphs, want = [], []
    for b, (k, v, q), out, w in sets:
        b.c.store(k, v, b.d_table, b.d_lengths, b.d_starts)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, weights=w)
        g.replay()
        want.append((out.clone(), w.clone()))
        graphs.append(g)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (b, x, out, w), (o, y) in zip(sets, want):
        assert torch.equal(out, o) and torch.equal(w, y)


def test_another_stream(world):
    """On a stream that is not the current one, behind work that is still running there."""
    b, (k, v, q), out, w = decode_setup(world, [1500, 700], room=1504)
    b.c.store(k, v, b.d_table, b.d_lengths, b.d_starts)
    b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, weights=w)
    want = out.clone(), w.clone()
    s = torch.cuda.Stream()
    late = torch.zeros_like(q)
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        a = torch.randn(2048, 2048, device="cuda")
        for _ in range(10):
            a = a @ a * 1e-3
        late.copy_(q)
    b.c.attend(late, out, b.d_table, b.d_lengths, b.d_starts, weights=w, stream=s)
    s.synchronize()
    assert torch.equal(out, want[0]) and torch.equal(w, want[1])


def test_lengths_and_rows_are_cut(world):
    """A sequence longer than max_length counts as that long, one with more rows than max_rows loses the last of them, a negative
    length is none, one beyond its table's room is cut to it."""
    b, (k, v, q), out, w = decode_setup(world, [90, -3, 1000])
    lse = world.full((3, 8), 44.0, torch.float32)
    b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, max_length=70, lse=lse)
    got, got_lse = world.get(out), world.get(lse)
    assert (got[1] == 0).all() and np.isneginf(got_lse[1]).all()
    for s, n in ((0, 70), (2, 70)):
        lengths = torch.tensor([n], dtype=torch.int32, device="cuda")
        o, z = torch.zeros_like(out[:1]), torch.zeros_like(lse[:1])
        b.c.attend(q[s:s + 1], o, b.d_table[s:s + 1], lengths, b.d_starts[:2], lse=z)
        close(world.get(z)[0], got_lse[s], np.full(8, 1e-4), "lse")
        close(world.get(o)[0], got[s], np.full(got[s].shape, 2 * ref.EPS["bf16"] * np.abs(got[s]).max()), "out")
    b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, max_rows=0, lse=lse)
    assert torch.equal(out, world.put(got, torch.bfloat16)), "rows were written that max_rows leaves out"


def test_places_beyond_32_bits(world):
    """Pages, rows, heads and weights more than 2^32 bytes (and elements) apart."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB")
    heads, d, page = 2, 64, 32
    size = world.cache.page_bytes(heads, d, page)
    n_pages = (5 << 30) // size
    pages = torch.empty(n_pages, size, dtype=torch.uint8, device="cuda")
    c = world.cache.Cache(pages, heads, d, page)
    table = torch.full((1, (1 << 25) + 8), -1, dtype=torch.int32, device="cuda")     # room for 2^30 slots
    last = [n_pages - 1, 0, n_pages - 2]
    table[0, :3] = torch.tensor(last, dtype=torch.int32)
    far = 1 << 31                                                                    # elements between rows
    store = torch.empty(far + 200, dtype=torch.bfloat16, device="cuda"), torch.empty(far + 200, dtype=torch.bfloat16, device="cuda")
    k, v = (x.as_strided((2, heads, d), (far, d, 1)) for x in store)
    rng = np.random.default_rng(5)
    for n in range(0, 70, 2):
        for x in (k, v):
            x.copy_(torch.from_numpy(rng.standard_normal((2, heads, d)).astype(np.float32)))
        lengths = torch.tensor([n + 2], dtype=torch.int32, device="cuda")
        starts = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
        c.store(k, v, table, lengths, starts)
    few = ref.Pages(world.get(pages[[last[0], last[1], last[2]]]), heads, d, page)
    held = [[few.rows(np.arange(3), h, 70) for h in range(heads)]]
    back = torch.empty_like(store[0]), torch.empty_like(store[0])
    bk, bv = (x.as_strided((2, heads, d), (far, d, 1)) for x in back)
    c.load(bk, bv, table, lengths, starts)
    for h in range(heads):
        for got, want in ((bk, held[0][h][0][68:]), (bv, held[0][h][1][68:])):
            close(world.get(got[:, h]), want, (ref.EPS["bf16"] + 2.0 ** -24) * np.abs(want), "rows back")
    most = 1 << 30
    weights = torch.empty(1, heads, most, dtype=torch.float32, device="cuda")
    q = store[0].as_strided((2, heads, d), (far, d, 1))
    out = store[1].as_strided((2, heads, d), (far, d, 1))
    qs = world.get(q)
    c.attend(q, out, table, lengths, starts, weights=weights, max_length=most)
    part = [[[x[i] for x in per] for per in held] for i in range(3)]
    want, _, w, tol, _, tol_w = ref.attention(qs, *part, [70], [0, 2], 1, d ** -0.5, True, 0, "bf16")
    close(world.get(out), want, tol, "out")
    close(world.get(weights[:, :, :70])[0], w[0], tol_w[0], "weights")
    to_lengths = world.full((1,), 0, torch.int32)
    _, kept = c.evict(weights, table, lengths, 20, torch.tensor([[n_pages - 5]], dtype=torch.int32, device="cuda"), to_lengths, max_length=most)
    stays = ref.evict([world.get(weights[0, :, :70]).astype(np.float32)], [70], 20, 0, 0)
    assert world.get(kept)[0].tolist() == stays
    new, old = ref.Pages(world.get(pages[[n_pages - 5]]), heads, d, page), few
    for h in range(heads):
        for i, slot in enumerate(stays[h]):
            for x, y in zip(new.row(0, h, i)[:2], old.row(slot // 32, h, slot % 32)[:2]):
                for a, e in zip(x, y):
                    assert np.array_equal(a, e)


def test_eviction_of_long_sequences(world):
    """More slots than a workgroup holds in registers: weights read again for each pass."""
    check_evict(world, [20000, 16385, 100], 1, 64, 128, 900, 4, 64)
    check_evict(world, [20000], 1, 64, 128, 130, 0, 0, make=lambda rng, shape: np.floor(rng.random(shape) * 3))


def test_eviction_outside_graphs_leaves_inputs(world):
    b, x, out, w = decode_setup(world, [90, 5, 64])
    w.uniform_()
    keep = w.clone(), b.d_lengths.clone(), b.d_table.clone()
    to_lengths = world.full((3,), 0, torch.int32)
    to = torch.tensor([[b.free[0]], [b.free[1]], [-1]], dtype=torch.int32, device="cuda")   # the third has nowhere to go
    old = b.pages.clone()
    to_w, kept = b.c.evict(w, b.d_table, b.d_lengths, 20, to, to_lengths)
    assert torch.equal(w, keep[0]) and torch.equal(b.d_lengths, keep[1]) and torch.equal(b.d_table, keep[2])
    assert to_lengths.tolist() == [20, 5, 20]
    same = (old == b.pages).all(1)
    assert same.tolist() == [p not in b.free[:2] for p in range(b.n_pages)]


def test_nothing_held(world):
    """No slots at all, by the table or by max_length: rows see nothing, no weight is written, nothing stays."""
    b, (k, v, q), out, w = decode_setup(world, [90, 5, 64])
    none = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    for table, kw in ((none, {}), (b.d_table, dict(max_length=0))):
        out.fill_(7.0)
        lse, w = world.full((3, 8), 7.0, torch.float32), world.full((3, 2, 1), 33.0, torch.float32)
        b.c.attend(q, out, table, b.d_lengths, b.d_starts, lse=lse, weights=w, **kw)
        assert (out == 0).all() and torch.isneginf(lse).all() and (w == 33).all()
        to_lengths = world.full((3,), 9, torch.int32)
        to_w, kept = b.c.evict(w, table, b.d_lengths, 20, torch.tensor([[b.free[0]]] * 3, dtype=torch.int32, device="cuda"), to_lengths, **kw)
        assert to_lengths.tolist() == [0, 0, 0] and (kept == -1).all() and (to_w == 0).all()
    old = b.pages.clone()
    b.c.store(k, v, none, b.d_lengths, b.d_starts)
    k.fill_(7.0)
    b.c.load(k, v, none, b.d_lengths, b.d_starts)
    assert torch.equal(old, b.pages) and (k == 7).all()


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("group", [2, 20])
def test_queries_that_are_none(world, type_, group):
    """A row of NaNs gives NaNs and nothing else changes; a row of zeros the mean."""
    def edit(q):
        q[0, 0] = float("nan")
        q[1, :, ::2] = 0.0
        q[2] = 0.0
    check_attend(world, [90, 40], [2, 2], 1, group, 64, 32, type_, q_edit=edit)


@pytest.mark.parametrize("type_", ["bf16", "f32"])
@pytest.mark.parametrize("q_scale", [1e20, 1e-25])
@pytest.mark.parametrize("group", [2, 20])
def test_attend_large_and_small_queries(world, group, q_scale, type_):
    check_attend(world, [70, 300], [2, 1], 1, group, 128, 32, type_, q_scale=q_scale)


def test_memory_for_a_stream_comes_from_it(world):
    """Scratch memory and results that a call makes for another stream are that stream's."""
    seen = []

    class Watched(torch.Tensor):
        def new_empty(self, *a, **kw):
            seen.append(torch.cuda.current_stream())
            return self.as_subclass(torch.Tensor).new_empty(*a, **kw)

    b, (k, v, q), out, w = decode_setup(world, [1500, 700], room=1504)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    b.c.attend(q.as_subclass(Watched), out, b.d_table, b.d_lengths, b.d_starts, weights=w, stream=s)
    to = torch.tensor([[b.free[0]], [b.free[1]]], dtype=torch.int32, device="cuda")
    to_lengths = world.full((2,), 0, torch.int32)
    torch.cuda.synchronize()
    b.c.evict(w.as_subclass(Watched), b.d_table, b.d_lengths, 20, to, to_lengths, stream=s)
    torch.cuda.synchronize()
    assert seen == [s, s, s]
