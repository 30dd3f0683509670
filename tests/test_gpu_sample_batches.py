"""b200_sample on batches so large that rows are read by small clusters, against the definition
(test_gpu_sample.py) and against the same rows sampled one at a time.

Sums are whole numbers, so a row's token does not depend on the batch it comes in: those
comparisons are exact.
"""
import numpy as np
import pytest
import torch

from test_gpu_sample import check, draw, logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [524289, 800128])
@pytest.mark.parametrize("rows", [60, 370, 500])
def test_long_16_bit_rows_of_equal_logits(cuda, kind, vocab, rows):
    """Nearly all tokens of a long row in one bin of the histogram: their weights' sum is far
    past 32 bits."""
    x = torch.zeros((1, vocab), device=cuda, dtype=kind)
    x[0, vocab // 3] = 8.6875
    x = x.expand(rows, -1)
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    pick = [0, 1, rows // 3, rows // 2, rows - 1]
    for args in ((1.0, 0, 0.5, 0.0), (1.0, 0, 0.9, 0.0), (1.0, vocab - 5, 0.5, 0.0)):
        got = draw(x, *args, u)
        check(x[pick], *args, u[pick], got[pick])
        assert int(got[pick[2]]) == int(draw(x[:1], *args, u[pick[2]])[0])
