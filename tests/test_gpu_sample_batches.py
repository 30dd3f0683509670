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


def settings(n, seed):
    rng = np.random.default_rng(seed)
    return (rng.choice([0.0, 0.6, 1.0, 1.7], n).astype(np.float32), rng.choice([0, 0, 5, 50, 700, 5000], n).astype(np.int32),
            rng.choice([0.0, 0.5, 0.9, 0.99, 1.0], n).astype(np.float32),
            rng.choice([0.0, 0.0, 0.02, 1.0], n).astype(np.float32)), rng.random(n).astype(np.float32)


def alone(x, args, u, row):
    return int(draw(x[row:row + 1], *[v[row] for v in args], u[row])[0])


@pytest.mark.parametrize("kind,vocab", [(torch.float32, 151936), (torch.float32, 151935), (torch.bfloat16, 200001),
                                        (torch.float16, 700000)])
@pytest.mark.parametrize("rows", [120, 400])
def test_large_batches(cuda, kind, vocab, rows):
    """Mixed settings; random, flat and stepped rows; rows that start at any element."""
    x = torch.empty((rows, vocab), device=cuda, dtype=kind)
    for r in range(0, rows, 40):
        x[r:r + 40] = logits(40, vocab, kind, rows + r)
    i = torch.arange(vocab, device=cuda)
    x[7] = 1.5
    x[8] = (i * 7919 % 5).to(kind)
    x[9] = (i * 7919 % 97).to(kind) * 0.25
    args, u = settings(rows, vocab + rows)
    got = draw(x, *args, u)
    pick = sorted({7, 8, 9} | set(np.random.default_rng(1).integers(0, rows, 24).tolist()))
    for r in pick:
        assert int(got[r]) == alone(x, args, u, r), (r, [v[r] for v in args], u[r])
    few = pick[:6] + [7, 8, 9]
    check(x[few], *[v[few] for v in args], u[few], got[few])


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


@pytest.mark.parametrize("vocab", [151936, 2 ** 20])
def test_min_p_of_a_few_units(cuda, vocab):
    """min_p of less than two units of 2^-40 keeps the tokens whose weight is one unit: they hold
    the last vocab - 1 units of the sum."""
    x = torch.full((1, vocab), -27.6, device=cuda)  # floor(2^40 e^-27.6) = 1
    x[0, 0] = 0.0
    u = np.float32(1) - np.float32(2.0 ** -24)  # 2^16 units before the end
    want = int(np.floor(np.float64(u) * (2.0 ** 40 + vocab - 1)) - 2.0 ** 40) + 1
    assert want > 0
    for min_p in (0.0, 0.95e-12, 1.2e-12, 1.7e-12, 1.8e-12):
        got = draw(x, 1.0, None, None, min_p, u)
        assert int(got[0]) == want, (min_p, int(got[0]), want)
