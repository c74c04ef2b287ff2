"""8-bit rows where counts are large and scales close: more units than an index of threads holds, the norm's factor to its last bits."""
import pytest
import torch

import my_own_cnn_b200 as b2q

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_reads_past_2_27_rows(cuda_lib, dtype):
    """A row that is not aligned is a warp's: 2^27 of them have 2^32 threads."""
    t = 2 ** 27 + 9
    rows = b2q.S8Rows(torch.zeros(t, 16, dtype=torch.int8, device="cuda"), torch.ones(t, device="cuda"), 1)
    marks = [0, 1, 2 ** 27 - 1, 2 ** 27, 2 ** 27 + 1, t - 1]
    rows.codes[marks, 0] = torch.arange(1, 7, dtype=torch.int8, device="cuda")
    y = rows.dequantize(dtype)
    assert y[marks, 0].tolist() == [1, 2, 3, 4, 5, 6]
    y[marks] = 0
    assert not y.any()
