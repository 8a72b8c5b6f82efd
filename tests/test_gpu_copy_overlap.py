"""Row copies whose source and destination share rows: left out, with a status bit, since the units of a move have no order."""
import numpy as np
import pytest
import torch

from gpu_util import dev, host, say
from test_gpu_share import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("row", [34, 136, 544])
@pytest.mark.parametrize("n", [2, 5, 16, 300])
def test_moves_over_themselves(gpu, row, n):
    say(f"copy: moves over themselves, rows of {row}, {n} of them")
    rng = np.random.default_rng(n)
    y = rng.integers(0, 256, (5 * n + 40, row), np.uint8)
    for by in sorted({1, n // 2, n - 1, n, n + 1}):
        for s, d in ((n + 3, n + 3 + by), (n + 3 + by, n + 3)):
            over = by < n
            x = [dev(y), dev(y[::-1])]
            gpu.device_status()
            # between a move that stands by itself and one onto itself, which is none (but 3 rows are more than max_rows of 2)
            gpu.paged_copy(x, i32([(0, 4 * n + 10, n), (s, d, n), (4 * n + 2, 4 * n + 2, 3)]), n)
            assert gpu.device_status() == (gpu.DEVERR_SET_ROWS_INDEX if over or n < 3 else 0)
            for a, b in zip(x, (y, y[::-1])):
                want = b.copy()
                want[4 * n + 10:5 * n + 10] = b[:n]
                if not over:
                    want[d:d + n] = b[s:s + n]
                assert np.array_equal(host(a), want), (by, s, d)
