"""The 4-bit cache's kernels and entry points on the CPU execution model (tests/emu), against the definition in 64 bits."""
import numpy as np
import pytest
import torch

from cache_world import (World, check_attend, check_evict, check_run, check_store, huge_values, late_nan, late_nan_key, tiny_keys,
                         tiny_values)


@pytest.fixture(scope="module")
def world(emu_sources):
    from conftest import ROOT, _load_file
    import os
    harness = _load_file("emu_harness", os.path.join(ROOT, "tests", "emu", "harness.py"))
    binding = harness.load_cache_binding(emu_sources.build_cache_library())
    device = harness.EmuTorch(binding.lib())
    return World(binding, device, lambda: None, lambda shape, dtype: device.empty(shape, dtype))


@pytest.fixture(autouse=True)
def _release(world):
    yield
    world.device.release()


@pytest.mark.parametrize("lengths,rows,heads,d,page,type_", [
    ([1], [1], 1, 64, 32, "bf16"),
    ([40, 33], [7, 33], 2, 128, 32, "f16"),
    ([5, 0, 70], [2, 0, 3], 3, 64, 64, "f32"),
    ([3], [5], 1, 256, 32, "bf16"),          # more rows than slots: the first ones have none
])
def test_store_and_load(world, lengths, rows, heads, d, page, type_):
    check_store(world, lengths, rows, heads, d, page, type_, padding=2)


def test_store_strided_and_bad_pages(world):
    check_store(world, [40], [40], 2, 64, 32, "bf16", strided=True)
    check_store(world, [70, 33], [70, 33], 1, 64, 32, "f32", bad_pages=[(0, 1, -1), (1, 0, 1 << 30)])


def blocks(rng, shape):
    """Blocks that are hard to hold: constant ones, borders hit exactly, huge, tiny, NaNs and infinities."""
    x = rng.standard_normal(shape)
    x = x.reshape(-1, 32)
    x[0::9] = 0.0
    x[1::9] = 3.5
    x[2::9] = np.arange(32) % 31 * 0.5                       # every border of step 1
    x[3::9] *= 1e6
    x[4::9] = x[4::9] * 1e-7
    x[5::9, 3] = np.nan
    x[6::9, 4] = -np.inf
    x[7::9] = -1000.0 + x[7::9] * 1e-3
    x[8::9] = -np.abs(x[8::9]) * 1e-30
    return x.reshape(shape)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
def test_store_hard_blocks(world, type_):
    check_store(world, [20], [20], 1, 128, 32, type_, make=blocks)


@pytest.mark.parametrize("lengths,rows,heads,group,d,page,type_,kw", [
    ([1], [1], 1, 1, 64, 32, "bf16", {}),
    ([33, 64], [1, 2], 2, 3, 64, 32, "bf16", {}),
    ([70], [20], 1, 2, 64, 64, "f32", dict(padding=3)),
    ([300], [1], 1, 4, 128, 64, "bf16", {}),                          # several parts joined
    ([40, 0, 5], [3, 0, 7], 1, 2, 64, 32, "f16", {}),                 # rows in front of slot 0 see nothing
    ([50], [6], 1, 3, 64, 32, "f32", dict(causal=False)),
    ([90], [9], 1, 2, 64, 32, "bf16", dict(window=11)),
    ([90], [4], 1, 2, 64, 32, "f32", dict(window=1, causal=False)),
    ([40], [2], 1, 1, 256, 32, "f32", {}),
    ([64], [1], 2, 2, 128, 32, "f16", dict(strided=True)),
    ([96], [3], 1, 2, 64, 32, "f32", dict(bad_pages=[(0, 1, -1)], weights=True)),
    ([70, 20], [5, 1], 2, 3, 64, 32, "f32", dict(weights=True, window=40)),
    ([70, 20], [5, 0], 1, 3, 64, 32, "bf16", dict(weights=True, in_place=True, tight=False)),
    ([35], [2], 1, 20, 64, 32, "f16", dict(weights=True, prior=False)),
])
def test_attend(world, lengths, rows, heads, group, d, page, type_, kw):
    check_attend(world, lengths, rows, heads, group, d, page, type_, **kw)


# Many columns: records unpacked once for several tiles of sixteen, and what falls back from there.
@pytest.mark.parametrize("lengths,rows,heads,group,d,page,type_,kw", [
    ([100], [33], 1, 2, 64, 32, "bf16", {}),                                    # 5 tiles
    ([70, 33], [40, 2], 1, 4, 64, 32, "f16", dict(padding=1)),                  # 10 tiles, of the second sequence one
    ([40], [20], 1, 2, 256, 32, "bf16", dict(strided=True)),
    ([300], [9], 1, 2, 64, 32, "f16", dict(window=30)),                         # parts
    ([90], [9], 1, 4, 64, 32, "bf16", dict(causal=False, weights=True)),
    ([130], [10], 1, 3, 64, 32, "bf16", dict(edit=huge_values)),
    ([130], [10], 1, 3, 64, 32, "f16", dict(edit=tiny_values, weights=True)),
    ([130], [10], 1, 3, 64, 32, "bf16", dict(edit=tiny_keys)),
    ([70], [8], 1, 3, 64, 32, "bf16", dict(edit=late_nan)),
    ([70], [8], 1, 3, 64, 32, "f16", dict(edit=late_nan_key, weights=True)),
    ([100], [10], 1, 3, 64, 32, "bf16", dict(bad_pages=[(0, 1, 99)])),
    ([320], [300], 1, 1, 64, 32, "bf16", dict(window=40)),                      # a tile sees a part of what its parts are cut from
    ([320], [300], 1, 1, 64, 32, "bf16", dict(window=40, edit=huge_values)),
])
def test_attend_many_columns(world, lengths, rows, heads, group, d, page, type_, kw):
    check_attend(world, lengths, rows, heads, group, d, page, type_, **kw)


@pytest.mark.parametrize("type_", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("edit", [huge_values, tiny_values, tiny_keys, late_nan, late_nan_key])
def test_attend_hard_rows(world, edit, type_):
    check_attend(world, [100], [3], 1, 2, 64, 32, type_, edit=edit)


@pytest.mark.parametrize("type_", ["bf16", "f32"])
@pytest.mark.parametrize("q_scale", [1e20, 1e-25])
@pytest.mark.parametrize("group", [2, 20])
def test_attend_large_and_small_queries(world, group, q_scale, type_):
    check_attend(world, [70], [2], 1, group, 64, 32, type_, q_scale=q_scale)


@pytest.mark.parametrize("type_", ["bf16", "f32"])
def test_operators_together(world, type_):
    check_run(world, type_=type_)


@pytest.mark.parametrize("lengths,heads,d,page,keep,first,recent", [
    ([50], 1, 64, 32, 20, 2, 5),
    ([70, 10, 0], 2, 128, 32, 33, 0, 33),
    ([40], 1, 64, 32, 40, 1, 1),
    ([33], 1, 256, 32, 1, 0, 0),
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
    check_evict(world, [60, 45], 2, 64, 32, 21, 3, 4, make=odd, bad_pages=[(0, 1, 5000)])
