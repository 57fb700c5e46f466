"""CPU: BlockTables refuses sizes that its kernels refuse, before it allocates."""
import pytest

from paceserve_b200 import cabi
from paceserve_b200.block_tables import MAX_REQUESTS, BlockTables
from tests.test_cabi import _expect


def test_more_rows_than_a_step_takes():
    with pytest.raises(RuntimeError, match="at most 8192 requests"):
        BlockTables(8193, 4, 16, 8, 100, "cuda")
    # the kernels' own limit
    lib = cabi.load()
    call = lambda n: lib.pace_release_pages(None, 4, 4, None, None, n, 16, None, 4, None, None, None, None)  # noqa: E731
    _expect(call(MAX_REQUESTS), cabi.PACE_ERR_INVALID_ARGUMENT, "null pointer")
    _expect(call(MAX_REQUESTS + 1), cabi.PACE_ERR_TOO_LARGE, "at most 8192")


def test_other_sizes():
    with pytest.raises(RuntimeError, match="all sizes"):
        BlockTables(8, 4, 0, 8, 100, "cuda")
    with pytest.raises(RuntimeError, match="past 32 bits"):
        BlockTables(8192, 1 << 18, 16, 8, 100, "cuda")
    with pytest.raises(RuntimeError, match="CUDA device"):
        BlockTables(8, 4, 16, 8, 100, "cpu")
