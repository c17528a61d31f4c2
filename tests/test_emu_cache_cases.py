"""Further cases of the 4-bit cache on the CPU execution model."""
import pytest

from cache_cases import (FAR, FAR_QUERIES, check_lse_without_and_with_weights, check_rows_left_out, check_store_exact, check_weights_of_large_scores,
                         close_keys, close_queries, hard_blocks)
from cache_world import check_attend, check_evict, check_store
from test_emu_cache import _release, world  # noqa: F401

# sequences' rows, max_rows, rows the arrays hold
LEFT_OUT = [([300], 5, None), ([300], None, 8), ([300, 3], 2, 302)]


@pytest.mark.parametrize("causal,window", [(False, 9), (True, 9), (False, 0), (True, 0)])
@pytest.mark.parametrize("rows,max_rows,hold", LEFT_OUT)
@pytest.mark.parametrize("group,type_", [(1, "f32"), (1, "bf16"), (9, "bf16")])   # (the last: many columns)
def test_rows_left_out(world, rows, max_rows, hold, causal, window, group, type_):  # noqa: F811
    check_rows_left_out(world, [400, 40][:len(rows)], rows, 1, group, 64, 32, type_, causal, window, max_rows, hold)


# (float16 results do not reach that far)
@pytest.mark.parametrize("edit", FAR)
@pytest.mark.parametrize("lengths,rows,group,d,type_,kw", [
    ([70], [2], 2, 64, "f32", {}), ([70], [2], 2, 64, "bf16", {}),
    ([300], [1], 1, 128, "f32", {}), ([300], [1], 1, 128, "bf16", dict(weights=True)),     # parts joined
    ([100], [9], 3, 64, "bf16", {}), ([100], [9], 3, 64, "bf16", dict(causal=False, window=20)),   # many columns
])
def test_attend_far_values(world, edit, lengths, rows, group, d, type_, kw):  # noqa: F811
    check_attend(world, lengths, rows, 1, group, d, 32, type_, edit=edit, **kw)


@pytest.mark.parametrize("seed", [0, 1])
def test_store_decides_exactly(world, seed):  # noqa: F811
    check_store_exact(world, hard_blocks(seed, 40))


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


@pytest.mark.parametrize("n", [65, 130])
def test_many_sequences(world, n):  # noqa: F811
    """More than a wave looks at together when it finds its rows' sequence; some hold nothing, some get nothing."""
    lengths = [(7 * i + i // 5) % 4 for i in range(n)]
    rows = [min(x, (3 * i) % 3) for i, x in enumerate(lengths)]
    check_store(world, lengths, rows, 1, 64, 32, "bf16", padding=1)
    check_attend(world, lengths, rows, 1, 2, 64, 32, "bf16", weights=True)
    check_evict(world, lengths, 1, 64, 32, 2, 1, 0)
