"""Further cases of the 4-bit cache on the GPU."""
import numpy as np
import pytest
import torch

from cache_cases import (FAR, FAR_QUERIES, check_lse_without_and_with_weights, check_rows_left_out, check_store_exact, check_weights_of_large_scores,
                         close_keys, close_queries, hard_blocks)
from cache_world import Batch, check_attend, check_evict, check_store, close
from test_emu_cache_cases import LEFT_OUT
from test_gpu_cache import world  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal,window", [(False, 9), (True, 9), (False, 0), (True, 0)])
@pytest.mark.parametrize("rows,max_rows,hold", LEFT_OUT)
@pytest.mark.parametrize("group,d,type_", [(1, 64, "f32"), (4, 128, "f16"), (9, 64, "bf16"), (20, 256, "bf16")])
def test_rows_left_out(world, rows, max_rows, hold, causal, window, group, d, type_):  # noqa: F811
    check_rows_left_out(world, [1300, 40][:len(rows)], rows, 1, group, d, 32, type_, causal, window, max_rows, hold)


@pytest.mark.parametrize("edit", FAR)
@pytest.mark.parametrize("lengths,rows,group,d,type_,kw", [
    ([70], [2], 2, 64, "f32", {}), ([70], [2], 2, 256, "bf16", {}),
    ([1300, 64], [1, 1], 1, 128, "f32", {}), ([1300], [1], 1, 128, "bf16", dict(weights=True)),         # parts joined
    ([200], [9], 3, 128, "bf16", {}), ([200, 90], [40, 3], 3, 64, "bf16", dict(causal=False, window=20)),   # many columns
])
def test_attend_far_values(world, edit, lengths, rows, group, d, type_, kw):  # noqa: F811
    check_attend(world, lengths, rows, 1, group, d, 32, type_, edit=edit, **kw)


@pytest.mark.parametrize("seed", [0, 1])
def test_store_decides_exactly(world, seed):  # noqa: F811
    check_store_exact(world, hard_blocks(seed, 400))


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scale", [1.0, -1.0, 0.5, 4.0])
@pytest.mark.parametrize("rows,group", [(1, 2), (10, 3)])
def test_large_scores_close_together(world, rows, group, scale, type_):  # noqa: F811
    check_attend(world, [250], [rows], 1, group, 64, 32, type_, scale=scale, edit=close_keys, q_edit=close_queries)


@pytest.mark.parametrize("type_", ["bf16", "f32"])   # (float16 queries do not reach that far)
@pytest.mark.parametrize("kw", FAR_QUERIES)
@pytest.mark.parametrize("lengths,rows,group", [([40], [1], 2), ([100], [9], 3), ([300], [2], 3)])
def test_largest_queries_and_scales(world, lengths, rows, group, kw, type_):  # noqa: F811
    check_attend(world, lengths, rows, 1, group, 64, 32, type_, **kw)


@pytest.mark.parametrize("type_", ["bf16", "f32"])
@pytest.mark.parametrize("q_scale", [1e6, 1e9, 1e20, 1e36])
@pytest.mark.parametrize("rows,group", [(1, 3), (7, 4)])
def test_weights_of_large_scores(world, rows, group, q_scale, type_):  # noqa: F811
    check_weights_of_large_scores(world, rows, group, type_, q_scale)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("d", [64, 256])
def test_lse_without_and_with_weights(world, d, type_):  # noqa: F811
    check_lse_without_and_with_weights(world, type_, d)


def test_many_long_sequences(world):  # noqa: F811
    """So many that a workgroup for each would take more than 128 records: their parts are others than those of a sequence alone, what they give is
    the same but for roundings."""
    n, heads, d, page = 64, 8, 64, 64
    lengths = [4200 - 61 * (i % 7) * (i % 9) for i in range(n)]
    b = Batch(world, lengths, [1] * n, heads, d, page, seed=5)
    b.fill()
    assert world.cache.lib() and b.c.scratch_bytes(n, heads, n, b.table.shape[1], torch.bfloat16, max_rows=1, max_length=4200, lse=True) == n * heads * 16 * 2 * (d + 2) * 4
    q = world.put(b.rng.standard_normal((n, heads, d)).astype(np.float32), torch.bfloat16)
    out, lse = world.full((n, heads, d), 0.0, torch.bfloat16), world.full((n, heads), 0.0, torch.float32)
    b.c.attend(q, out, b.d_table, b.d_lengths, b.d_starts, max_rows=1, max_length=4200, lse=lse)
    one, one_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for s in range(n):
        b.c.attend(q[s:s + 1], one[s:s + 1], b.d_table[s:s + 1], b.d_lengths[s:s + 1], b.d_starts[:2], lse=one_lse[s:s + 1])
    # (the same scores in the same waves' arithmetic: sums of 4200 terms, then roundings of out)
    close(world.get(lse), world.get(one_lse), np.full((n, heads), 2 * 4200 * 2.0 ** -24), "lse")
    got, want = world.get(out), world.get(one)
    close(got, want, np.full(got.shape, 2 * 2.0 ** -8 * np.abs(want).max()), "out")


def test_selection_near_2_to_31_slots(world):  # noqa: F811
    """The longest sequence that a table can hold: weights counted over it, then selected from its far end as from its front."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    most = (1 << 31) - 96
    pages = world.cache.new_pages(2, 1, 64, 32)
    c = world.cache.Cache(pages, 1, 64, 32)
    table = torch.full((1, most // 32), -1, dtype=torch.int32, device="cuda")      # (no page: nothing to see, zeros to move)
    lengths, starts = world.put(np.array([most], np.int32)), world.put(np.array([0, 1], np.int32))
    weights = torch.full((1, 1, most), 33.0, device="cuda")
    q, out, lse = world.full((1, 1, 64), 1.0, torch.bfloat16), world.full((1, 1, 64), 7.0, torch.bfloat16), world.full((1, 1), 7.0, torch.float32)
    c.attend(q, out, table, lengths, starts, lse=lse, weights=weights)
    assert (out == 0).all() and torch.isneginf(lse).all()
    assert not weights[0, 0, :1000].any() and not weights[0, 0, -100000:].any() and float(weights.sum()) == 0.0
    far = [5, 16383, 16384, 1 << 30, most - 16385, most - 96, most - 4]
    for i, slot in enumerate(far):
        weights[0, 0, slot] = 1.0 + i
    to_lengths = world.full((1,), 0, torch.int32)
    to_weights, kept = c.evict(weights, table, lengths, 12, world.full((1, 1), 1, torch.int32), to_lengths, first=2, recent=2)
    want = sorted([0, 1, 2] + far + [most - 2, most - 1])      # (one more place than weights: the first of the zeros)
    assert to_lengths.tolist() == [12] and kept[0, 0].tolist() == want
    assert to_weights[0, 0].tolist() == [0.0, 0.0, 0.0] + [1.0 + i for i in range(7)] + [0.0, 0.0]


@pytest.mark.parametrize("n", [65, 129, 1500])
def test_many_sequences(world, n):  # noqa: F811
    """More than a wave looks at together when it finds its rows' sequence; some hold nothing, some get nothing."""
    lengths = [(7 * i + i // 5) % 4 for i in range(n)]
    rows = [min(x, (3 * i) % 3) for i, x in enumerate(lengths)]
    check_store(world, lengths, rows, 1, 64, 32, "bf16", padding=1)
    check_attend(world, lengths, rows, 1, 2, 64, 32, "bf16", weights=True)
    check_evict(world, lengths, 1, 64, 32, 2, 1, 0)


def test_most_sequences(world):  # noqa: F811
    """65535 sequences of a row each: what is stored is loaded again, and a single slot's attention is its value."""
    n = 65535
    pages = world.cache.new_pages(n, 1, 64, 32)
    c = world.cache.Cache(pages, 1, 64, 32)
    table = torch.randperm(n, device="cuda").to(torch.int32)[:, None].contiguous()
    lengths, starts = torch.ones(n, dtype=torch.int32, device="cuda"), torch.arange(n + 1, dtype=torch.int32, device="cuda")
    k = (torch.randint(0, 16, (n, 1, 64), device="cuda") * 0.5).bfloat16()
    v = (torch.randint(0, 16, (n, 1, 64), device="cuda") - 7.0).bfloat16()
    k[:, :, ::32], k[:, :, 1::32], v[:, :, ::32], v[:, :, 1::32] = 0, 7.5, -7, 8       # (steps of 1/2 and 1: held exactly)
    c.store(k, v, table, lengths, starts)
    back = torch.zeros_like(k), torch.zeros_like(v)
    c.load(*back, table, lengths, starts)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    out = torch.zeros_like(v)
    c.attend(k, out, table, lengths, starts, max_rows=1, max_length=1)
    assert torch.equal(out, v)
    to_lengths = torch.zeros(n, dtype=torch.int32, device="cuda")
    more = torch.cat([pages, torch.empty_like(pages)])
    c = world.cache.Cache(more, 1, 64, 32)
    to = table + n
    weights, kept = c.evict(torch.rand(n, 1, 32, device="cuda"), table, lengths, 1, to, to_lengths)
    assert (to_lengths == 1).all() and not kept.any()
    c.load(*back, to, to_lengths, starts)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)


@pytest.mark.parametrize("type_,kw", [("bf16", dict(weights=True)), ("f32", dict(edit=FAR[1])), ("f16", dict(window=15000))])
def test_many_parts(world, type_, kw):  # noqa: F811
    """One long sequence, whose parts are more than those that join them at a time."""
    check_attend(world, [20011], [1], 1, 3, 64, 64, type_, **kw)


def test_many_parts_of_many_columns(world):  # noqa: F811
    check_attend(world, [9001], [9], 1, 4, 64, 64, "bf16", window=6000)
