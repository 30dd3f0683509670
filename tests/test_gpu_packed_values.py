"""b200_flash_attn_packed on values that are no numbers, against the same formulas in float64.

16-bit types: the bounds of test_gpu_batch.py.
"""
import math

import pytest
import torch

import b200infer as B
from test_gpu_batch import DT, check, cumulative, gen, packed_exact

pytestmark = pytest.mark.gpu

# every way a 16-bit call is cut: (heads, query lengths, key lengths); in each, every row
# sees at least the first 128 keys of its sequence
CUTS = {
    "halves": ((4, 2, 128), [64], [400]),
    "parts": ((4, 2, 128), [64], [3100]),
    "one_slot": ((16, 8, 128), [64] * 20, [200] * 20),
    "two_tiles": ((16, 8, 64), [2432], [2700]),
}


def inputs(seed, heads, ql, kl, kind):
    Hq, Hkv, D = heads
    g = gen(seed)
    return [torch.randn((n, h, D), device="cuda", generator=g).to(DT[kind])
            for n, h in ((sum(ql), Hq), (sum(kl), Hkv), (sum(kl), Hkv))]


def scores_at_any_position(kind, cut):
    """A key whose K holds a NaN, or whose score is +inf, leaves no number in the rows that see
    it, wherever in the tile it lies; -inf scores count for nothing. V is finite throughout."""
    heads, ql, kl = CUTS[cut]
    Hq, Hkv, D = heads
    G = Hq // Hkv
    q, k, v = inputs(31, heads, ql, kl, kind)
    q[..., 0] = 1.0
    cu_q, cu_k = cumulative(ql), cumulative(kl)
    want, w = packed_exact(q, k, v, ql, kl)
    n = ql[0]  # rows of the first sequence, which alone sees the keys below
    for at in range(40, 48):
        for value, d in ((math.nan, 3), (math.inf, 0)):
            bad = k.clone()
            bad[at, 0, d] = value
            got = B.flash_attn_packed(q, bad, v, cu_q, cu_k)
            assert torch.isnan(got[:n, :G].double()).all(), (at, value)
            check(got[:, G:], want[:, G:], w[:, G:], kind, True)
            if len(ql) > 1:
                check(got[n:], want[n:], w[n:], kind, True)
    some = k.clone()
    some[40:48, 0, 0] = -math.inf
    want, w = packed_exact(q, some, v, ql, kl)
    check(B.flash_attn_packed(q, some, v, cu_q, cu_k), want, w, kind, True)


def rows_with_scores_of_minus_inf_alone(kind, ql, kl):
    """No weight is left: zeros, as for a row without keys."""
    heads = (16, 8, 128)
    q, k, v = inputs(32, heads, ql, kl, kind)
    q[..., 0] = 1.0
    n, m = ql[0], kl[0]
    k[:m, 0, 0] = -math.inf
    got = B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl))
    assert (got[:n, :2] == 0).all()
    want, w = packed_exact(q, torch.where(torch.isfinite(k), k, 0), v, ql, kl)
    check(got[:, 2:], want[:, 2:], w[:, 2:], kind, True)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("cut", list(CUTS))
def test_nan_and_inf_scores_at_any_position(cuda, kind, cut):
    scores_at_any_position(kind, cut)


ROWS = {"short": ([6], [40]), "halves": ([6], [400]), "parts": ([3], [3100]), "one_slot": ([64] * 20, [200] * 20),
        "causal": ([130], [130])}


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("lens", list(ROWS))
def test_rows_with_scores_of_minus_inf_alone(cuda, kind, lens):
    rows_with_scores_of_minus_inf_alone(kind, *ROWS[lens])


def test_f32_few_keys_with_scores_of_minus_inf_alone(cuda):
    rows_with_scores_of_minus_inf_alone("f32", *ROWS["short"])
