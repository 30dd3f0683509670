"""b200_flash_attn_packed on values that are no numbers, and on magnitudes that differ
within a key tile, against the same formulas in float64.

16-bit types: the bounds of test_gpu_batch.py. F32, per output element: operands and
weights hold at least 22 bits, so a score moves by at most 2^-21 of scale sum |q_d k_d|
(S below, the largest over the keys a row sees), a weight by as much, relative, and once more
through the softmax's sum; the weights' own bits, their exponential and the sums' rounding
add less than 2^-20. Together (2^-20 S + 2^-20) of sum_j p_j |v_jd|: the output column's own
magnitude, so neither other columns nor keys that a row does not see count.
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


# ---------------------------------------------------------------------------
# F32: magnitudes

def sums(q, k, v, past):
    """(n, Hq, D) over (m, Hkv, D): output, sum p |v| and S in float64."""
    n, Hq, D = q.shape
    m, Hkv, _ = k.shape
    seen = torch.arange(m, device=q.device)[None] <= past + torch.arange(n, device=q.device)[:, None]
    out = torch.zeros((n, Hq, D), dtype=torch.float64, device=q.device)
    size, S = torch.zeros_like(out), torch.zeros((n, Hq, 1), dtype=torch.float64, device=q.device)
    for h in range(Hq):
        g = h // (Hq // Hkv)
        a, b, x = q[:, h].double(), k[:, g].double(), v[:, g].double()
        p = torch.softmax((a @ b.T / math.sqrt(D)).masked_fill(~seen, -math.inf), -1)
        out[:, h], size[:, h] = p @ x, p @ x.abs()
        S[:, h, 0] = (a.abs() @ b.abs().T / math.sqrt(D)).masked_fill(~seen, 0.0).amax(1)
    return out, size, S


def check_f32(got, q, k, v, past, rows=slice(None)):
    want, size, S = (t[rows] for t in sums(q, k, v, past))
    assert torch.isfinite(got[rows]).all()
    worst = float(((got[rows].double() - want).abs() / ((2.0 ** -20 * S + 2.0 ** -20) * size)).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("cut", list(CUTS))
def test_f32_nan_and_inf_scores_at_any_position(cuda, cut):
    scores_at_any_position("f32", cut)


@pytest.mark.parametrize("lens", ["halves", "parts", "one_slot", "causal"])
def test_f32_rows_with_scores_of_minus_inf_alone(cuda, lens):
    rows_with_scores_of_minus_inf_alone("f32", *ROWS[lens])


LAYOUTS = {"g2": (16, 8, 128), "g2d64": (8, 4, 64), "g3": (6, 2, 128), "g16": (16, 1, 128)}


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("big", [1e4, 1e8, 1e12, 1e20, 3e38])
@pytest.mark.parametrize("where", ["k", "v", "both"])
def test_f32_hidden_keys_of_any_finite_value(cuda, layout, big, where):
    """Rows before a large finite K or V row do not see it, although it lies in their tile."""
    q, k, v = inputs(33, LAYOUTS[layout], [200], [200], "f32")
    kk, vv = k.clone(), v.clone()
    for at in (100, 190):
        if where != "v":
            kk[at] *= big / 4
        if where != "k":
            vv[at] *= big / 4
    got = B.flash_attn_packed(q, kk, vv, cumulative([200]))
    check_f32(got, q, k, v, 0, slice(0, 100))


def magnitudes_within_a_tile(layout, power, case):
    """Columns or rows of a tile that differ by 2^power: each output keeps its own digits."""
    T = 300
    q, k, v = inputs(34, LAYOUTS[layout], [T], [T], "f32")
    D = q.shape[2]
    odd = torch.arange(D, device="cuda") % 2 == 1
    if case == "v_columns":
        v[..., odd] *= 2.0 ** -power
    elif case == "k_columns":  # what K loses Q brings back
        k[..., odd] *= 2.0 ** -power
        q[..., odd] *= 2.0 ** power
    elif case == "v_rows":  # later keys are larger
        v *= 2.0 ** (power * torch.arange(T, device="cuda") / T)[:, None, None]
    else:
        k *= 2.0 ** (-power * (torch.arange(T, device="cuda") % 2))[:, None, None]
    check_f32(B.flash_attn_packed(q, k, v, cumulative([T])), q, k, v, 0)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("power", [10, 20, 30])
@pytest.mark.parametrize("case", ["v_columns", "k_columns", "v_rows", "k_rows"])
def test_f32_magnitudes_within_a_tile(cuda, layout, power, case):
    magnitudes_within_a_tile(layout, power, case)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("power", [12, 13, 15])
@pytest.mark.parametrize("case", ["v_columns", "k_columns", "v_rows", "k_rows"])
def test_f32_magnitudes_that_one_exponent_holds(cuda, layout, power, case):
    magnitudes_within_a_tile(layout, power, case)


@pytest.mark.parametrize("layout", list(LAYOUTS))
def test_f32_large_elements_in_different_columns(cuda, layout):
    """Q and K rows of magnitude 2^70 whose products are of order one."""
    T = 150
    q, k, v = inputs(35, LAYOUTS[layout], [T], [T], "f32")
    q[..., 0] *= 2.0 ** 70
    k[..., 0] *= 2.0 ** -70
    q[..., 1] *= 2.0 ** -70
    k[..., 1] *= 2.0 ** 70
    check_f32(B.flash_attn_packed(q, k, v, cumulative([T])), q, k, v, 0)


def test_f32_tiny_operands_and_a_large_scale(cuda):
    """Exponents of Q and K far below what one F32 factor holds: all scores are next to 0."""
    T = 150
    q, k, v = inputs(36, (4, 2, 64), [T], [T], "f32")
    got = B.flash_attn_packed(q * 1e-30, k * 1e-30, v, cumulative([T]), scale=1e30)
    check_f32(got, torch.zeros_like(q), k, v, 0)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("lens", [(3, 5000), (40, 1500)])
def test_f32_one_odd_tile_among_many(cuda, layout, lens):
    """A call cut into parts of the keys, one tile of which needs more bits than the others."""
    n, m = lens
    q, k, v = inputs(37, LAYOUTS[layout], [n], [m], "f32")
    q[..., 0] = 2.0 ** -40
    k[..., 0] *= 0.5
    k[m // 2, :, 0] = 2.0 ** 40
    check_f32(B.flash_attn_packed(q, k, v, cumulative([n]), cumulative([m])), q, k, v, m - n)


@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("at", [40, 250, 398])
def test_f32_visible_infinite_values(cuda, layout, at):
    """An infinite V element makes its column infinite in the rows that see it, and no other."""
    n, m = 9, 400
    q, k, v = inputs(38, LAYOUTS[layout], [n], [m], "f32")
    want = v.clone()
    v[at, :, 5] = math.inf
    v[at, :, 6] = -math.inf
    got = B.flash_attn_packed(q, k, v, cumulative([n]), cumulative([m]))
    see = slice(max(0, at - (m - n)), n)
    assert (got[see, :, 5] == math.inf).all() and (got[see, :, 6] == -math.inf).all()
    rest = [d for d in range(q.shape[2]) if d not in (5, 6)]
    exact, size, S = sums(q, k, want, m - n)
    bound = (2.0 ** -20 * S + 2.0 ** -20) * size
    assert ((got.double() - exact).abs() <= bound)[..., rest].all()
    if see.start:
        assert ((got.double() - exact).abs() <= bound)[:see.start].all()


# ---------------------------------------------------------------------------
# offsets out of range

@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("T", [50, 170])
@pytest.mark.parametrize("cu_q,cu_k,good", [
    ([0, 20, 60, 50], None, [(0, 20)]), ([0, 20, 500, 700], None, [(0, 20)]), ([-5, 20, 30, 50], None, [(20, 30), (30, 50)]),
    ([0, 20, 30, 50], [0, 20, 900, 50], [(0, 20)]), ([0, 20, 20, 50], [0, 20, -7, 50], [(0, 20)]),
    ([30, 20, 10, 0], None, [])], ids=["past", "far", "negative", "keys", "keys_of_an_empty_one", "descending"])
def test_bad_offsets_leave_zeros(cuda, kind, T, cu_q, cu_k, good):
    """Rows that no sequence with offsets in range covers are zeros; the others are as ever."""
    heads = (4, 2, 64)
    q, k, v = inputs(39, heads, [T], [T], kind)
    scale = lambda cu: None if cu is None else torch.tensor(  # noqa: E731
        [c * T // 50 for c in cu], dtype=torch.int32, device=cuda)
    out = torch.full_like(q, math.nan)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    B.flash_attn_packed(q, k, v, scale(cu_q), scale(cu_k), out=out, status=status)
    assert int(status) == 2  # B200_DEV_BAD_POSITION
    left = torch.ones(T, dtype=torch.bool, device=cuda)
    for a, b in good:
        a, b = a * T // 50, b * T // 50
        want, w = packed_exact(q[a:b], k[a:b], v[a:b], [b - a], [b - a])
        check(out[a:b], want, w, kind, True)
        left[a:b] = False
    assert (out[left] == 0).all()
