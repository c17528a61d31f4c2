"""The 4-bit cache on the GPU, against the definition in 64 bits (tests/cache_reference.py)."""
import numpy as np
import pytest
import torch

import __graft_entry__ as entry
from cache_world import TYPES, Batch, World, check_attend, check_evict, check_store

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
