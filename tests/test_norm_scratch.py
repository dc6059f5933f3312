"""The scratch of the norms' gradient goes by the rows there are: three sums a CTA that has rows and one a stretch of rows, not those of a full GPU."""
import pytest

from mytorch_b200.backends.cuda.env import LIBRARY_PATH, NativeError, _binding


@pytest.mark.parametrize("rows", [1, 2, 7, 100])
@pytest.mark.parametrize("c", [8, 96, 1023, 1024, 8192, 16384, 1 << 20])
def test_few_rows_take_little(rows, c):
    _binding.load(LIBRARY_PATH, NativeError)
    need = _binding.add_rms_norm_workspace_bytes(rows, c)
    assert 12 * c <= need <= 4 * 4 * rows * c + 16


@pytest.mark.parametrize("c", [8, 96, 1024, 8192, 20000])
def test_many_rows_take_no_more_than_a_full_gpu(c):
    _binding.load(LIBRARY_PATH, NativeError)
    needs = [_binding.add_rms_norm_workspace_bytes(rows, c) for rows in (0, 1, 50, 1000, 10 ** 5, 10 ** 7, 2 ** 31 - 1)]
    assert needs == sorted(needs) and needs[0] > 0 and needs[-1] == needs[-2]
