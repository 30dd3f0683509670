"""Batched serving attention (b200_flash_attn_packed, b200_paged_kv_append,
b200_flash_attn_paged_batch) against the same formulas in float64.

Bounds, per output element with `want` exact:
  F32: 1e-5 of |want| + RMS(want), the bar of the F32 kernels (test_gpu_ops.py).
  F16 / BF16, unit roundoff u = 2^-11 / 2^-8: the output's one rounding, u |want|; where P is
  rounded before the second product, its terms p_j v_j move by at most u each, independently:
  a standard deviation of at most u / sqrt(3) of W = sqrt(sum (p_j v_j)^2), allowed 4 u W
  (seven deviations); the F32 bar for the rest; 2^-25 for F16 outputs below its normals.
"""
import math

import numpy as np
import pytest
import torch

import b200infer as B

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LAYOUTS = {"g2": (16, 8, 128), "g4": (32, 8, 128), "g2d64": (8, 4, 64), "g1": (3, 3, 64), "g3": (6, 2, 128),
           "g7": (7, 1, 64), "g16": (16, 1, 128), "g20": (20, 1, 64)}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def exact(q, k, v, past, scale=None):
    """(n, Hq, D) over (m, Hkv, D), row i sees keys 0 .. past + i: output and W in float64."""
    n, Hq, D = q.shape
    m, Hkv, _ = k.shape
    out = torch.zeros((n, Hq, D), dtype=torch.float64, device=q.device)
    w = torch.zeros_like(out)
    seen = torch.arange(m, device=q.device)[None] <= past + torch.arange(n, device=q.device)[:, None]
    some = seen.any(1) if m else torch.zeros(n, dtype=torch.bool, device=q.device)
    if not bool(some.any()):
        return out, w
    for h in range(Hq):
        g = h // (Hq // Hkv)
        s = q[:, h].double() @ k[:, g].double().T * (scale or 1 / math.sqrt(D))
        p = torch.softmax(s.masked_fill(~seen, -math.inf)[some], -1)
        # a hidden key counts for nothing whatever its row holds
        vv = torch.where(seen[some].any(0)[:, None], v[:, g].double(), 0.0)
        out[some, h] = p @ vv
        w[some, h] = torch.sqrt(p.square() @ vv.square())
    return out, w


def check(got, want, w, kind, rounded_p):
    assert torch.isfinite(got.double()).all()
    u = UNIT[kind]
    rms = float(want.square().mean().sqrt())
    bound = u * want.abs() + (4 * u if rounded_p else 4 * u * u) * w + 1e-5 * (want.abs() + rms) + 2.0 ** -25
    err = (got.double() - want).abs()
    worst = float((err / bound).max()) if err.numel() else 0.0
    assert worst <= 1.0, worst


def cumulative(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def packed_exact(q, k, v, ql, kl, scale=None):
    outs, ws, a, b = [], [], 0, 0
    for n, m in zip(ql, kl):
        o, w = exact(q[a:a + n], k[b:b + m], v[b:b + m], m - n, scale)
        outs.append(o), ws.append(w)
        a, b = a + n, b + m
    return torch.cat(outs), torch.cat(ws)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("lens", [([1], [1]), ([37], [37]), ([64, 0, 1, 129, 63], [64, 0, 1, 129, 63]),
                                  ([5, 1, 70], [133, 400, 70]), ([40, 3, 0, 9], [7, 0, 12, 9])],
                         ids=["one", "short", "ragged", "chunked", "empty_rows"])
def test_packed(cuda, kind, layout, lens):
    Hq, Hkv, D = LAYOUTS[layout]
    ql, kl = lens
    g = gen(len(layout) * 100 + sum(ql))
    q = torch.randn((sum(ql), Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    got = B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl))
    want, w = packed_exact(q, k, v, ql, kl)
    check(got, want, w, kind, True)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64"])
def test_packed_long(cuda, kind, layout):
    Hq, Hkv, D = LAYOUTS[layout]
    ql = [1333, 2, 700, 129, 128, 257]
    kl = [1333, 2, 1900, 129, 1000, 257]
    g = gen(5)
    q = torch.randn((sum(ql), Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = (torch.randn((sum(kl), Hkv, D), device=cuda, generator=g) + 0.5).to(DT[kind])
    got = B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl))
    want, w = packed_exact(q, k, v, ql, kl)
    check(got, want, w, kind, True)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g2d64", "g16"])
@pytest.mark.parametrize("lens", [([1], [5000]), ([3, 40, 1, 0], [6100, 45, 1, 7]), ([200, 9], [1700, 4003])],
                         ids=["one", "short_beside_long", "chunks"])
def test_packed_few_rows_long_contexts(cuda, kind, layout, lens):
    """Few query tiles and many keys, so the keys of a tile are shared out among CTAs, some of
    which get none; hidden keys that are no numbers."""
    Hq, Hkv, D = LAYOUTS[layout]
    ql, kl = lens
    g = gen(17)
    q = torch.randn((sum(ql), Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = (torch.randn((sum(kl), Hkv, D), device=cuda, generator=g) + 0.5).to(DT[kind])
    want, w = packed_exact(q, k, v, ql, kl)
    for fill in (0, 0x7C, 0xFF):  # what a workspace held before is never read
        n = B.lib().b200_flash_attn_packed_workspace_bytes(len(ql), sum(ql), sum(kl), D, Hq, Hkv, list(DT).index(kind))
        ws = torch.full((n,), fill, dtype=torch.uint8, device=cuda)
        check(B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl), workspace=ws), want, w, kind, True)
    k[kl[0] - 1], v[kl[0] - 1] = math.nan, math.inf  # seen by the first sequence's last row alone
    got = B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl))
    rows = [i for i in range(sum(ql)) if i != ql[0] - 1]
    if rows:
        check(got[rows], want[rows], w[rows], kind, True)
    assert not torch.isfinite(got[ql[0] - 1].double()).any()


@pytest.mark.parametrize("kind", list(DT))
def test_packed_strides_scale_and_growing_scores(cuda, kind):
    """Q, K and V as views of one projection output, an output inside a wider tensor, a
    given scale, and scores that grow along the keys (the running maximum moves)."""
    Hq, Hkv, D, ql = 4, 2, 128, [200, 77]
    T = sum(ql)
    g = gen(9)
    qkv = torch.randn((T, Hq + 2 * Hkv, D), device=cuda, generator=g)
    qkv[:, Hq:Hq + Hkv] *= torch.linspace(0.2, 12, T, device=cuda)[:, None, None]
    qkv = qkv.to(DT[kind])
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    wide = torch.full((T, 2 * Hq, D), 7.0, device=cuda, dtype=DT[kind])
    B.flash_attn_packed(q, k, v, cumulative(ql), scale=0.11, out=wide[:, ::2])
    want, w = packed_exact(q, k, v, ql, ql, 0.11)
    check(wide[:, ::2], want, w, kind, True)
    assert (wide[:, 1::2] == 7).all()


@pytest.mark.parametrize("kind", list(DT))
def test_packed_other_layouts(cuda, kind):
    """Head-major K and V, one KV row shared by all heads (stride 0), token-strided Q."""
    Hq, Hkv, D, ql = 8, 4, 64, [260, 31]
    T = sum(ql)
    g = gen(10)
    q = torch.randn((T, 2, Hq, D), device=cuda, generator=g).to(DT[kind])[:, 1]
    kv = torch.randn((2, Hkv, T, D), device=cuda, generator=g).to(DT[kind])
    k, v = kv[0].transpose(0, 1), kv[1].transpose(0, 1)
    one = torch.randn((T, 1, D), device=cuda, generator=g).to(DT[kind]).expand(T, Hkv, D)
    for kk, vv in ((k, v), (one, v), (one, one)):
        got = B.flash_attn_packed(q, kk, vv, cumulative(ql))
        want, w = packed_exact(q, kk, vv, ql, ql)
        check(got, want, w, kind, True)


@pytest.mark.parametrize("kind", list(DT))
def test_packed_many_short_sequences(cuda, kind):
    """More sequences than a warp looks at in one round, many of them empty."""
    Hq, Hkv, D = 4, 2, 64
    ql = [(i * 5) % 7 if i % 3 else 0 for i in range(150)] + [200]
    kl = [n + (i * 11) % 40 if n else 0 for i, n in enumerate(ql)]
    g = gen(12)
    q = torch.randn((sum(ql), Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    want, w = packed_exact(q, k, v, ql, kl)
    check(B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl)), want, w, kind, True)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", [(32, 8, 64), (16, 8, 128), (24, 8, 64)], ids=["g4d64", "g2d128", "g3d64"])
def test_packed_many_tiles_with_hidden_keys(cuda, kind, layout):
    """So many query tiles that a CTA takes two at a time; each sequence's last key is no number and
    its last row alone sees it."""
    Hq, Hkv, D = layout
    ql, kl = [1500, 3, 1100], [1500, 130, 1171]
    g = gen(19)
    q = torch.randn((sum(ql), Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    want, w = packed_exact(q, k, v, ql, kl)
    check(B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl)), want, w, kind, True)
    ends = [i - 1 for i in cumulative(kl)[1:].tolist()]
    k[ends], v[ends] = math.inf, math.nan
    got = B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl))
    last = [i - 1 for i in cumulative(ql)[1:].tolist()]
    rows = [i for i in range(sum(ql)) if i not in last]
    check(got[rows], want[rows], w[rows], kind, True)
    assert not torch.isfinite(got[last].double()).any()


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", [(32, 8, 64), (16, 8, 128), (24, 8, 64)], ids=["g4d64", "g2d128", "g3d64"])
@pytest.mark.parametrize("lens", [([2300, 1211], [2300, 1900]), ([1500, 0, 3, 900, 130] * 7, [1501, 9, 3, 900, 100] * 7),
                                  ([90] * 40, [140] * 40)], ids=["two_tiles", "many", "more_than_lanes"])
def test_packed_many_tiles_of_any_lengths(cuda, kind, layout, lens):
    """Long contexts in pairs of tiles, and more sequences than a warp has lanes, some of them with
    rows that see no key; the first sequence's last key is no number."""
    Hq, Hkv, D = layout
    ql, kl = lens
    g = gen(23)
    q = torch.randn((sum(ql), Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((sum(kl), Hkv, D), device=cuda, generator=g).to(DT[kind])
    want, w = packed_exact(q, k, v, ql, kl)
    check(B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl)), want, w, kind, True)
    k[kl[0] - 1], v[kl[0] - 1] = math.inf, math.nan
    got = B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl))
    rows = [i for i in range(sum(ql)) if i != ql[0] - 1]
    check(got[rows], want[rows], w[rows], kind, True)
    assert not torch.isfinite(got[ql[0] - 1].double()).any()


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_packed_hidden_keys_of_any_value(cuda, kind, bad):
    """Non-finite K and V rows that a query does not see leave its row as it is: later keys of
    its own sequence, another sequence's keys, rows outside every sequence."""
    Hq, Hkv, D, ql = 4, 2, 128, [150, 90]
    g = gen(11)
    q = torch.randn((sum(ql) + 40, Hq, D), device=cuda, generator=g).to(DT[kind])
    k = torch.randn((sum(ql) + 40, Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((sum(ql) + 40, Hkv, D), device=cuda, generator=g).to(DT[kind])
    cu = cumulative(ql)
    clean = B.flash_attn_packed(q, k, v, cu)
    hidden = [140, 141, 239] + list(range(240, 280))
    k[hidden], v[hidden] = bad, bad
    got = B.flash_attn_packed(q, k, v, cu)
    rows = list(range(140)) + list(range(150, 239))
    assert torch.isfinite(got[rows].double()).all()
    want, w = packed_exact(q[:240], torch.where(torch.isfinite(k), k, 0)[:240], torch.where(torch.isfinite(v), v, 0)[:240],
                           ql, ql)
    check(got[rows], want[rows], w[rows], kind, True)
    check(clean[rows], want[rows], w[rows], kind, True)
    if not bad < 0:  # the rows that do see them: their weights are no numbers
        assert not torch.isfinite(got[141:150].double()).any() and not torch.isfinite(got[239].double()).any()


@pytest.mark.parametrize("kind", list(DT))
def test_packed_extreme_magnitudes(cuda, kind):
    """Rows of very different magnitudes: large values and tiny ones of the type."""
    Hq, Hkv, D, ql = 2, 1, 64, [130, 70]
    g = gen(13)
    big = 3e4 if kind == "f16" else 1e30
    small = 1e-4 if kind == "f16" else 1e-30
    q = torch.randn((200, Hq, D), device=cuda, generator=g)
    k = torch.randn((200, Hkv, D), device=cuda, generator=g)
    v = torch.rand((200, Hkv, D), device=cuda, generator=g) + 0.5
    v[:130] *= big / 2
    v[130:] *= small
    q, k, v = (t.to(DT[kind]) for t in (q, k, v))
    got = B.flash_attn_packed(q, k, v, cumulative(ql))
    want, w = packed_exact(q, k, v, ql, ql)
    check(got[:130].double() / big, want[:130] / big, w[:130] / big, kind, True)
    if kind == "f16":  # below its normals: steps of 2^-24
        assert (got[130:].double() - want[130:]).abs().max() <= 2.0 ** -11 * small * 2 + 2.0 ** -25
    else:
        check(got[130:].double() / small, want[130:] / small, w[130:] / small, kind, True)


def test_packed_bad_offsets_are_reported_not_followed(cuda):
    q = torch.randn((50, 4, 64), device=cuda)
    k = torch.randn((50, 2, 64), device=cuda)
    for cu in ([0, 20, 10, 50], [0, 20, 60, 70], [-5, 20, 30, 50]):
        cu = torch.tensor(cu, dtype=torch.int32, device=cuda)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        B.flash_attn_packed(q, k, k, cu, status=status)
        assert int(status) == 2  # B200_DEV_BAD_POSITION
        status.zero_()
        B.flash_attn_packed(q, k, k, torch.tensor([0, 20, 30, 50], dtype=torch.int32, device=cuda), cu, status=status)
        assert int(status) == 2


def test_packed_rows_outside_the_sequences_are_untouched(cuda):
    q = torch.randn((50, 4, 64), device=cuda)
    k = torch.randn((50, 2, 64), device=cuda)
    out = torch.full_like(q, 3.0)
    B.flash_attn_packed(q, k, k, torch.tensor([0, 17, 41], dtype=torch.int32, device=cuda), out=out)
    assert (out[41:] == 3).all() and not (out[:41] == 3).any()


# ---------------------------------------------------------------------------
# the paged cache

class Cache:
    """Pools of more blocks than the table names, in shuffled order, all NaN at first; K and V
    are two halves of one tensor (strided), or separate."""

    def __init__(self, lens, bt, Hkv, D, kind, seed, joint=False):
        per = [-(-n // bt) for n in lens]
        blocks = sum(per) + 3
        order = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
        self.table = torch.full((len(lens), max(max(per), 1) + 2), -1, dtype=torch.int32)
        for i, n in enumerate(per):
            self.table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.table = self.table.cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        nan = math.nan
        if joint:
            kv = torch.full((blocks, bt, 2, Hkv, D), nan, device="cuda", dtype=DT[kind])
            self.k, self.v = kv[:, :, 0], kv[:, :, 1]
        else:
            self.k = torch.full((blocks, bt, Hkv, D), nan, device="cuda", dtype=DT[kind])
            self.v = torch.full_like(self.k, nan)
        self.bt = bt

    def rows(self, s, n):
        j = torch.arange(n, device="cuda")
        b = self.table[s].long()[j // self.bt]
        return self.k[b, j % self.bt], self.v[b, j % self.bt]


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("bt", [1, 7, 16, 128])
@pytest.mark.parametrize("joint", [False, True])
def test_append(cuda, kind, bt, joint):
    """Three appends (a prompt, one step, another chunk) leave every sequence's rows in order
    and every other slot as it was."""
    Hkv, D = 3, 64
    rounds = [[33, 0, 1, 140], [1, 1, 1, 1], [0, 20, 5, 3]]
    final = [sum(r[s] for r in rounds) for s in range(4)]
    c = Cache(final, bt, Hkv, D, kind, bt, joint)
    g = gen(bt)
    kept = [[], [], [], []]
    done = [0, 0, 0, 0]
    for new in rounds:
        T = sum(new)
        qkv = torch.randn((T, 4 + 2 * Hkv, D), device=cuda, generator=g).to(DT[kind])
        k, v = qkv[:, 4:4 + Hkv], qkv[:, 4 + Hkv:]
        done = [a + b for a, b in zip(done, new)]
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        B.paged_kv_append(k, v, cumulative(new), torch.tensor(done, dtype=torch.int32, device=cuda), c.k, c.v, c.table,
                          status=status)
        assert int(status) == 0
        at = 0
        for s, n in enumerate(new):
            kept[s].append((k[at:at + n], v[at:at + n]))
            at += n
    used = 0
    for s, n in enumerate(final):
        k, v = c.rows(s, n)
        assert torch.equal(k, torch.cat([x[0] for x in kept[s]])) and torch.equal(v, torch.cat([x[1] for x in kept[s]]))
        used += n
    assert int((~torch.isnan(c.k[..., 0, 0])).sum()) == used and int((~torch.isnan(c.v[..., 0, 0])).sum()) == used


def test_append_many_sequences(cuda):
    n, bt = 2000, 4
    new = [(i * 7) % 4 for i in range(n)]
    c = Cache([max(x, 1) for x in new], bt, 1, 64, "f16", 3)
    T = sum(new)
    k = torch.arange(T, device=cuda, dtype=torch.float32)[:, None, None].expand(T, 1, 64).remainder(2048).half().contiguous()
    B.paged_kv_append(k, -k, cumulative(new), torch.tensor(new, dtype=torch.int32, device=cuda), c.k, c.v, c.table)
    at = 0
    got_k, got_v = c.k.cpu(), c.v.cpu()
    table = c.table.cpu()
    for s, m in enumerate(new):
        if m:
            assert torch.equal(got_k[table[s, 0], :m], k[at:at + m].cpu())
            assert torch.equal(got_v[table[s, 0], :m], -k[at:at + m].cpu())
        at += m


def test_append_reports_what_it_cannot_place(cuda):
    c = Cache([20, 20], 16, 2, 64, "f32", 1)
    k = torch.randn((4, 2, 64), device=cuda)
    for lens, cu in (([20, 100], [0, 2, 4]), ([1, 20], [0, 2, 4]), ([20, 20], [0, 2, 3]), ([20, 20], [1, 2, 4])):
        c.k.fill_(math.nan)
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        B.paged_kv_append(k, k, torch.tensor(cu, dtype=torch.int32, device=cuda),
                          torch.tensor(lens, dtype=torch.int32, device=cuda), c.k, c.v, c.table, status=status)
        assert int(status) == 2
        assert int((~torch.isnan(c.k[..., 0, 0])).sum()) <= 3


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("bt,lens", [(16, [1]), (16, [301]), (7, [5, 0, 64, 65, 63, 1, 200]), (128, [1000, 3, 129]),
                                     (1, [33, 2]), (100, [4097])],
                         ids=["one", "single", "ragged", "pages128", "pages1", "long"])
def test_decode(cuda, kind, layout, bt, lens):
    Hq, Hkv, D = LAYOUTS[layout]
    g = gen(bt + sum(lens))
    c = Cache(lens, bt, Hkv, D, kind, 7, joint=bt == 128)
    k = torch.randn((sum(lens), Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((sum(lens), Hkv, D), device=cuda, generator=g).to(DT[kind])
    B.paged_kv_append(k, v, cumulative(lens), c.lens, c.k, c.v, c.table)
    q = torch.randn((len(lens), Hq, D), device=cuda, generator=g).to(DT[kind])
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens, status=status)
    assert int(status) == 0
    again = B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens)
    assert torch.equal(got, again)
    want, w = packed_exact(q, k, v, [1] * len(lens), lens)
    for i, n in enumerate(lens):
        if n == 0:
            want[i], w[i] = 0, 0
    check(got, want, w, kind, False)


@pytest.mark.parametrize("kind", list(DT))
def test_decode_many_ragged(cuda, kind):
    """More pairs than CTAs and one long sequence among short ones; strided q and out."""
    Hq, Hkv, D, bt = 8, 4, 64, 16
    lens = [(i * 37) % 90 for i in range(300)] + [9000]
    c = Cache(lens, bt, Hkv, D, kind, 7)
    g = gen(21)
    k = (torch.randn((sum(lens), Hkv, D), device=cuda, generator=g) * 2).to(DT[kind])
    v = torch.randn((sum(lens), Hkv, D), device=cuda, generator=g).to(DT[kind])
    B.paged_kv_append(k, v, cumulative(lens), c.lens, c.k, c.v, c.table)
    wide = torch.randn((len(lens), Hq + 3, D), device=cuda, generator=g).to(DT[kind])
    q = wide[:, 2:2 + Hq]
    out = torch.full((len(lens), Hq, 2 * D), 5.0, device=cuda, dtype=DT[kind])
    B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens, scale=0.2, out=out[..., :D])
    want, w = packed_exact(q, k, v, [1] * len(lens), lens, 0.2)
    for i, n in enumerate(lens):
        if n == 0:
            want[i], w[i] = 0, 0
    check(out[..., :D], want, w, kind, False)
    assert (out[..., D:] == 5).all()


def test_decode_past_2_31_bytes(cuda):
    """A pool whose byte offsets pass 32 bits: the last blocks are read where they are."""
    Hkv, D, bt = 8, 128, 64
    blocks = 2 ** 33 // (bt * Hkv * D * 2) + 5
    k = torch.zeros((blocks, bt, Hkv, D), device=cuda, dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    k[-2:] = torch.randn((2, bt, Hkv, D), device=cuda).bfloat16()
    v[-2:] = torch.randn((2, bt, Hkv, D), device=cuda).bfloat16()
    table = torch.tensor([[blocks - 1, blocks - 2]], dtype=torch.int32, device=cuda)
    lens = torch.tensor([100], dtype=torch.int32, device=cuda)
    q = torch.randn((1, 16, D), device=cuda).bfloat16()
    got = B.flash_attn_paged_batch(q, k, v, table, lens)
    kk = torch.cat([k[-1], k[-2]])[:100]
    vv = torch.cat([v[-1], v[-2]])[:100]
    want, w = exact(q, kk, vv, 99)
    check(got, want, w, "bf16", False)


@pytest.mark.parametrize("kind", list(DT))
def test_decode_bad_blocks_and_lengths(cuda, kind):
    """Keys of a block out of range are left out, a length past the table is cut; both reported."""
    Hq, Hkv, D, bt, lens = 8, 2, 128, 16, [100, 50]
    c = Cache(lens, bt, Hkv, D, kind, 2)
    g = gen(3)
    k = torch.randn((150, Hkv, D), device=cuda, generator=g).to(DT[kind])
    v = torch.randn((150, Hkv, D), device=cuda, generator=g).to(DT[kind])
    B.paged_kv_append(k, v, cumulative(lens), c.lens, c.k, c.v, c.table)
    q = torch.randn((2, Hq, D), device=cuda, generator=g).to(DT[kind])
    table = c.table.clone()
    table[0, 2] = 10 ** 6
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = B.flash_attn_paged_batch(q, c.k, c.v, table, c.lens, status=status)
    assert int(status) == 2
    keep = [j for j in range(100) if j // bt != 2]
    want0, w0 = exact(q[:1], k[keep], v[keep], len(keep) - 1)
    want1, w1 = exact(q[1:], k[100:], v[100:], 49)
    check(got[:1], want0, w0, kind, False)
    check(got[1:], want1, w1, kind, False)
    status.zero_()
    short = c.table[:, :2].contiguous()
    got = B.flash_attn_paged_batch(q, c.k, c.v, short, c.lens, status=status)
    assert int(status) == 2
    want0, w0 = exact(q[:1], k[:32], v[:32], 31)
    check(got[:1], want0, w0, kind, False)
    status.zero_()
    got = B.flash_attn_paged_batch(q, c.k, c.v, c.table, torch.tensor([-4, 50], dtype=torch.int32, device=cuda), status=status)
    assert int(status) == 2 and (got[0] == 0).all()
    check(got[1:], want1, w1, kind, False)


def test_calls_on_another_stream_and_in_a_graph(cuda):
    """The calls go to torch's current stream and can be captured; a replay sees new lengths."""
    Hq, Hkv, D, bt, lens = 8, 4, 64, 16, [90, 40]
    c = Cache([200, 200], bt, Hkv, D, "bf16", 2)
    k = torch.randn((130, Hkv, D), device=cuda).bfloat16()
    c.lens.copy_(torch.tensor(lens))
    B.paged_kv_append(k, k, cumulative(lens), c.lens, c.k, c.v, c.table)
    q = torch.randn((2, Hq, D), device=cuda).bfloat16()
    out = torch.zeros_like(q)
    ws = torch.empty(B.lib().b200_flash_attn_paged_batch_workspace_bytes(2, c.table.shape[1] * bt, D, Hq, Hkv, 2), dtype=torch.uint8, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    first = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        B.flash_attn_paged_batch(q, c.k, c.v, c.table, c.lens, out=out, workspace=ws)
    out.zero_()
    graph.replay()
    assert torch.equal(out, first)
    c.lens.copy_(torch.tensor([17, 40]))
    graph.replay()
    want, w = exact(q[:1], k[:17], k[:17], 16)
    check(out[:1], want, w, "bf16", False)
    assert torch.equal(out[1], first[1])


def test_refusals(cuda):
    q = torch.randn((10, 4, 64), device=cuda)
    k = torch.randn((10, 2, 64), device=cuda)
    cu = cumulative([10])
    for call in (lambda: B.flash_attn_packed(q.double(), k.double(), k.double(), cu),
                 lambda: B.flash_attn_packed(q, k.half(), k.half(), cu),
                 lambda: B.flash_attn_packed(q[:, :3], k, k, cu),
                 lambda: B.flash_attn_packed(q, k, k[:9], cu),
                 lambda: B.flash_attn_packed(q, k, k, cu.long()),
                 lambda: B.flash_attn_packed(q, k, k, cu.cpu()),
                 lambda: B.flash_attn_packed(q, k, k, cu, out=q[:5]),
                 lambda: B.flash_attn_packed(q.transpose(1, 2).contiguous().transpose(1, 2), k, k, cu),
                 lambda: B.flash_attn_paged_batch(q, k[None], k[None], cu[None], cu),
                 lambda: B.paged_kv_append(k, k[:5], cu, cu[:1], k[None], k[None], cu[None])):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(B.B200Error) as e:  # head_dim 32
        B.flash_attn_packed(q[..., :32].contiguous(), k[..., :32].contiguous(), k[..., :32].contiguous(), cu)
    assert e.value.status == 2
    odd = torch.randn(10 * 4 * 64 + 1, device=cuda)[1:].view(10, 4, 64)  # 4 bytes off a 16-byte boundary
    with pytest.raises(B.B200Error) as e:
        B.flash_attn_packed(odd, k, k, cu)
    assert e.value.status == 2
    # nothing to do
    assert B.flash_attn_packed(q[:0], k, k, cumulative([0])).shape == (0, 4, 64)
    B.paged_kv_append(k[:0], k[:0], cumulative([0]), cu[:1], k[None], k[None], cu[:1][None])
