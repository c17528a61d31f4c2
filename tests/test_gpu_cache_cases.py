"""Further cases of the 4-bit cache on the GPU."""
import pytest

from cache_cases import check_rows_left_out
from test_emu_cache_cases import LEFT_OUT
from test_gpu_cache import world  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal,window", [(False, 9), (True, 9), (False, 0), (True, 0)])
@pytest.mark.parametrize("rows,max_rows,hold", LEFT_OUT)
@pytest.mark.parametrize("group,d,type_", [(1, 64, "f32"), (4, 128, "f16"), (9, 64, "bf16"), (20, 256, "bf16")])
def test_rows_left_out(world, rows, max_rows, hold, causal, window, group, d, type_):  # noqa: F811
    check_rows_left_out(world, [1300, 40][:len(rows)], rows, 1, group, d, 32, type_, causal, window, max_rows, hold)
