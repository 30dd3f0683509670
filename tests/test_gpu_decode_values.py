"""b200_flash_attn_paged_batch on values that are no numbers, and at the end of 31 bits. Bounds: those of
test_gpu_batch.py, on the elements that are numbers."""
import math

import pytest
import torch

import b200infer as B
from test_gpu_batch import DT, LAYOUTS, Cache, check, cumulative, gen, packed_exact

pytestmark = pytest.mark.gpu


def cached(lens, layout, kind, bt, seed):
    Hq, Hkv, D = LAYOUTS[layout]
    c = Cache(lens, bt, Hkv, D, kind, seed)
    g = gen(seed)
    k, v = (torch.randn((sum(lens), Hkv, D), device="cuda", generator=g).to(DT[kind]) for _ in range(2))
    q = torch.randn((len(lens), Hq, D), device="cuda", generator=g).to(DT[kind])
    return c, q, k, v


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g2d64", "g7", "g16", "g20"])
@pytest.mark.parametrize("lens", [[1], [70, 300, 5], [9] * 150 + [2000]], ids=["one", "few", "many"])
def test_infinite_values(cuda, kind, layout, lens):
    """An infinite V element makes its column infinite, both signs in one column none; a NaN stays
    in its column. Other columns, and other sequences, are as ever."""
    c, q, k, v = cached(lens, layout, kind, 16, 41)
    want, w = packed_exact(q, k, v, [1] * len(lens), lens)
    ends = [sum(lens[:i + 1]) for i in range(len(lens))]
    # the first, a middle and the last key of the last sequence, whose weights are not small
    first, last = ends[-1] - lens[-1], ends[-1] - 1
    mid = (first + last) // 2
    k[[first, mid, last]] = 0
    v[first, :, 3] = math.inf
    v[last, :, 4] = -math.inf
    v[mid, :, 5] = math.nan
    v[first, :, 6], v[last, :, 6] = math.inf, -math.inf if last > first else math.inf
    want2, w2 = packed_exact(q[-1:], k[first:], torch.where(torch.isfinite(v), v, 0)[first:], [1], lens[-1:])
    B.paged_kv_append(k, v, cumulative(lens), c.lens, c.k, c.v, c.table)
    got = B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens)
    rest = [d for d in range(q.shape[2]) if d not in (3, 4, 5, 6)]
    check(got[-1:, :, rest], want2[..., rest], w2[..., rest], kind, False)
    assert (got[-1, :, 3] == math.inf).all() and (got[-1, :, 4] == -math.inf).all()
    assert torch.isnan(got[-1, :, 5].double()).all()
    assert torch.isnan(got[-1, :, 6].double()).all() if last > first else (got[-1, :, 6] == math.inf).all()
    if len(lens) > 1:
        check(got[:-1], want[:-1], w[:-1], kind, False)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g7", "g20"])
def test_nan_keys_and_scores_of_minus_inf(cuda, kind, layout):
    """A NaN in K leaves no number in the row; a row whose scores are all -inf is zero."""
    lens = [100, 60, 300]
    c, q, k, v = cached(lens, layout, kind, 7, 42)
    q[..., 0] = 1.0
    want, w = packed_exact(q, k, v, [1] * 3, lens)
    k[77, :, 1] = math.nan
    k[100:160, :, 0] = -math.inf
    B.paged_kv_append(k, v, cumulative(lens), c.lens, c.k, c.v, c.table)
    got = B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens)
    assert torch.isnan(got[0].double()).all() and (got[1] == 0).all()
    check(got[2:], want[2:], w[2:], kind, False)


@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_lengths_up_to_31_bits(cuda, kind):
    """One page of 2^31 - 1 positions that all share one row, and a length that reaches their end:
    cut at 2^31 - 257 and reported. The sums of equal rows of 1/2 are exact up to the join, whose
    rounding is far below half a unit of F16."""
    Hq, D = 2, 64
    row = torch.full((1, 1, 1, D), 0.5, device=cuda, dtype=DT[kind])
    pool = row.expand(1, 2 ** 31 - 1, 1, D)
    q = torch.randn((2, Hq, D), device=cuda).to(DT[kind])
    table = torch.zeros((2, 1), dtype=torch.int32, device=cuda)
    for length, code in ((2 ** 31 - 1, 2), (2 ** 31 - 257, 0), (2 ** 31 - 256, 2)):
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        lens = torch.tensor([length, 5], dtype=torch.int32, device=cuda)
        got = B.flash_attn_paged_batch(q, pool, pool, table, lens, status=status)
        assert int(status) == code
        assert (got.half() == 0.5).all()
