"""The 4-bit cache's binding: written tensors whose rows share memory are refused, others of any layout are not."""
import importlib
import random

import pytest
import torch

import __graft_entry__ as entry
from test_cache_abi import Call, cache  # noqa: F401


@pytest.fixture
def call(cache):  # noqa: F811
    return Call(cache)


def shared(rows, row, heads, head, d):
    """Whether two rows of d elements have one in common, by marking all of them."""
    seen = set()
    for i in range(rows):
        for j in range(heads):
            mine = set(range(i * row + j * head, i * row + j * head + d))
            if mine & seen:
                return True
            seen |= mine
    return False


def test_rows_that_share_memory(cache):  # noqa: F811
    rng = random.Random(3)
    found = [0, 0]
    for _ in range(3000):
        rows, heads, d = rng.randint(1, 5), rng.randint(1, 5), rng.randint(1, 6)
        row, head = rng.randint(0, 30), rng.randint(0, 30)
        want = shared(rows, row, heads, head, d)
        assert cache._share_memory(rows, row, heads, head, d) == want, (rows, row, heads, head, d)
        found[want] += 1
    assert min(found) > 300


def test_two_arrays_that_share_memory(cache):  # noqa: F811
    """Of one layout, the second `offset` elements behind the first; neither by itself."""
    rng = random.Random(4)
    found = [0, 0]
    while sum(found) < 1500:
        rows, heads, d = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 5)
        row, head, offset = rng.randint(0, 40), rng.randint(0, 40), rng.randint(-60, 60)
        if shared(rows, row, heads, head, d):
            continue
        first = {i * row + j * head + x for i in range(rows) for j in range(heads) for x in range(d)}
        want = any(x + offset in first for x in first)
        assert cache._meet(offset, rows, row, heads, head, d) == want, (rows, row, heads, head, d, offset)
        found[want] += 1
    assert min(found) > 150


def rows_of(buffer, strides, heads, offset=0):
    return buffer.as_strided((5, heads, 64), strides, offset)


MEMORY = torch.zeros(4000)


@pytest.mark.parametrize("strides", [(63, 400, 1), (128, 32, 1), (100, 64, 1), (64, 64, 1), (255, 64, 1), (256, 128, 1)])
def test_out_refused(call, strides):
    with pytest.raises(ValueError, match="own"):
        call.attend(out=rows_of(MEMORY, strides, 4))


@pytest.mark.parametrize("strides", [(256, 64, 1), (64, 320, 1), (300, 70, 1), (512, 64, 1), (130, 64 + 650, 1), (192, 704, 1)])
def test_out_taken(call, strides):
    with pytest.raises(ValueError, match="GPU"):
        call.attend(out=rows_of(MEMORY, strides, 4))


@pytest.mark.parametrize("strides,offset", [((127, 64, 1), 2000), ((128, 64, 1), 64), ((128, 64, 1), 639), ((256, 64, 1), 127), ((256, 64, 1), 65)])
def test_load_refused(call, strides, offset):
    with pytest.raises(ValueError, match="own"):
        call.load(k=rows_of(MEMORY, strides, 2), v=rows_of(MEMORY, strides, 2, offset))
    with pytest.raises(ValueError, match="own"):
        call.load(k=rows_of(MEMORY, strides, 2, offset), v=rows_of(MEMORY, strides, 2))


@pytest.mark.parametrize("strides,offset", [((128, 64, 1), 640), ((256, 64, 1), 128), ((256, 128, 1), 64), ((64, 640, 1), 320), ((300, 64, 1), 150)])
def test_load_taken(call, strides, offset):
    for a, b in ((0, offset), (offset, 0)):
        with pytest.raises(ValueError, match="GPU"):
            call.load(k=rows_of(MEMORY, strides, 2, a), v=rows_of(MEMORY, strides, 2, b))


def test_one_row_or_none(call):
    """Strides of a dimension that has one entry say nothing."""
    for n in (0, 1):
        with pytest.raises(ValueError, match="GPU"):
            call.attend(q=torch.zeros(n, 4, 64), out=torch.zeros(n, 4, 64).as_strided((n, 4, 64), (3, 64, 1)))
    with pytest.raises(ValueError, match="GPU"):
        call.store(k=rows_of(MEMORY, (0, 64, 1), 2), v=rows_of(MEMORY, (0, 64, 1), 2))      # (read alone)


def test_scratch_does_not_grow_with_the_lengths(cache):  # noqa: F811
    """Parts are cut for workgroups to be enough, at most eight a compute unit where there are not as many anyway: memory for them has a bound."""
    rng = random.Random(5)
    for _ in range(3000):
        heads, group, d = rng.choice([1, 2, 8, 32]), rng.choice([1, 4, 16, 40]), rng.choice([64, 128, 256])
        n, rows = rng.choice([1, 2, 7, 64, 300]), rng.choice([0, 1, 1, 5, 64, 3000, 20000])
        length = rng.choice([100, 5000, 131072, 1 << 20, 1 << 24])
        if n * rows * heads * group >= 1 << 31:
            continue
        type_ = rng.choice([torch.bfloat16, torch.float32])
        c = cache.Cache(torch.zeros(0, dtype=torch.uint8), heads, d, 64)
        need = c.scratch_bytes(n * rows, heads * group, n, -(-length // 64), type_, max_rows=rows, lse=True)
        tiles = -(-rows * group // 16)
        units = n * heads * tiles
        wide = type_ == torch.bfloat16 and tiles > 1
        # (a wide workgroup takes up to sixteen tiles)
        most = (2048 + units) * (16 if wide else 1) * 16 * (d + 2) * 4
        assert need <= most, (heads, group, d, n, rows, length, type_, need, most)
        if not wide and units >= 2048:
            assert need == 0, (heads, group, d, n, rows, length, type_, need)
