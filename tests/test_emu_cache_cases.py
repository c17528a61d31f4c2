"""Further cases of the 4-bit cache on the CPU execution model."""
import pytest

from cache_cases import check_rows_left_out
from test_emu_cache import _release, world  # noqa: F401

# sequences' rows, max_rows, rows the arrays hold
LEFT_OUT = [([300], 5, None), ([300], None, 8), ([300, 3], 2, 302)]


@pytest.mark.parametrize("causal,window", [(False, 9), (True, 9), (False, 0), (True, 0)])
@pytest.mark.parametrize("rows,max_rows,hold", LEFT_OUT)
@pytest.mark.parametrize("group,type_", [(1, "f32"), (1, "bf16"), (9, "bf16")])   # (the last: many columns)
def test_rows_left_out(world, rows, max_rows, hold, causal, window, group, type_):  # noqa: F811
    check_rows_left_out(world, [400, 40][:len(rows)], rows, 1, group, 64, 32, type_, causal, window, max_rows, hold)
