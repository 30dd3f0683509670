"""Shared-prefix attention with groups that fill tiles of rows (the tensor-core kernels of every type): values that are no
numbers, magnitudes that spread, hidden content, bad blocks, group sizes. Bounds as in test_gpu_shared.py."""
import math

import pytest
import torch

import b200infer as B
from test_gpu_shared import BAD_POSITION, DT, Batch, check, ints

pytestmark = pytest.mark.gpu

MANY = dict(prefix=[700, 130], seqs=[40, 11], lens=[(i * 29) % 60 for i in range(51)])


def many(layout, kind, seed, block=16):
    return Batch(MANY["prefix"], MANY["seqs"], MANY["lens"], block, layout, kind, seed)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64", "g16"])
def test_nan_keys(cuda, kind, layout):
    """A NaN in a prefix's key reaches its group's rows of that KV head alone, at any place in a tile."""
    b = many(layout, kind, 3)
    want, w = b.want()
    Hq, Hkv = b.q.shape[1], b.k.shape[2]
    G, h = Hq // Hkv, Hkv - 1
    for place in (0, 1, 130, 255, 698, 699):
        keep = b.k.clone()
        b.k[b.prefix_table[0, place // 16], place % 16, h, 7] = math.nan
        got = B.flash_attn_paged_shared(*b.args())
        odd = torch.zeros(got.shape[:2], dtype=torch.bool, device=cuda)
        odd[:40, h * G:] = True
        assert torch.isnan(got[odd]).all()
        check(got[~odd], want[~odd], w[~odd], kind)
        b.k = keep


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g2d64"])
def test_infinite_values(cuda, kind, layout):
    """An infinite element of V, of a prefix or of a sequence, makes that column of the rows that see it infinite."""
    b = many(layout, kind, 5)
    b.v[b.prefix_table[0, 2], 5, 1, 9] = math.inf
    b.v[b.prefix_table[1, 8], 1, 0, 3] = -math.inf
    b.v[b.table[7, 0], 0, 0, 60] = math.inf
    want, w = b.want()
    got = B.flash_attn_paged_shared(*b.args())
    fine = torch.isfinite(want)
    assert int((~fine).sum()) == (40 + 11 + 1) * b.q.shape[1] // b.k.shape[2]
    assert torch.equal(got.double()[~fine], want[~fine])
    w = torch.where(fine, w, 0.0)
    check(torch.where(fine, got.double(), 0.0).to(DT[kind]), torch.where(fine, want, 0.0), w, kind)


@pytest.mark.parametrize("kind", list(DT))
def test_scores_of_minus_infinity(cuda, kind):
    """Keys with scores of -inf count for nothing, and a row that has only such keys is zero."""
    b = Batch([256, 100], [40, 3], [(i * 7) % 5 for i in range(43)], 16, "g2", kind, 7)
    b.q.fill_(1.0)
    b.k[b.prefix_table[0].long()] = -math.inf
    got = B.flash_attn_paged_shared(*b.args())
    b.prefix[0] = 0
    want, w = b.want()
    check(got, want, w, kind)
    assert (got[0] == 0).all()


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64"])
@pytest.mark.parametrize("block", [16, 100, 7, 128, 1, 6])
def test_hidden_content(cuda, kind, layout, block):
    """What lies behind the ends, in last blocks and unused ones, does not count, whatever it is; blocks of any size."""
    b = many(layout, kind, 9, block)
    want = b.want()
    used = torch.zeros(b.k.shape[:2], dtype=torch.bool, device=cuda)
    for table, lens in ((b.prefix_table, b.prefix), (b.table, b.own)):
        for i, n in enumerate(lens):
            pos = torch.arange(n, device=cuda)
            used[table[i].long()[pos // block], pos % block] = True
    for bad in (math.nan, math.inf, -math.inf):
        b.k[~used] = bad
        b.v[~used] = bad
        check(B.flash_attn_paged_shared(*b.args()), *want, kind)


@pytest.mark.parametrize("layout", ["g2", "g2d64", "g16"])
def test_spread_magnitudes(cuda, layout):
    """F32 columns, keys and values whose magnitudes differ by far more than one exponent holds."""
    b = many(layout, "f32", 11)
    b.v[..., 3] *= 2.0 ** -40
    b.k[b.prefix_table[0, 5]] *= 2.0 ** -30
    b.v[b.prefix_table[0, 6]] *= 2.0 ** 30
    want, _ = b.want()
    got = B.flash_attn_paged_shared(*b.args())
    for rows in (slice(0, 40), slice(40, 51)):  # each group and column by its own magnitude
        for d in (3, 4):
            x, y = got[rows, :, d].double(), want[rows, :, d]
            assert ((x - y).abs() <= 1e-5 * (y.abs() + float(y.square().mean().sqrt()))).all()


@pytest.mark.parametrize("kind", list(DT))
def test_bad_blocks(cuda, kind):
    """A block out of range anywhere in a prefix clears its group's rows, whichever part of the keys it falls into."""
    b = many("g4", kind, 13)
    want, w = b.want()
    status = ints([0])
    for at in (0, 20, 43):
        keep = int(b.prefix_table[0, at])
        for bad in (-1, b.k.shape[0], 2 ** 31 - 1):
            b.prefix_table[0, at] = bad
            status.zero_()
            got = B.flash_attn_paged_shared(*b.args(), status=status)
            assert int(status) == BAD_POSITION and (got[:40] == 0).all()
            check(got[40:], want[40:], w[40:], kind)
        b.prefix_table[0, at] = keep
    status.zero_()
    check(B.flash_attn_paged_shared(*b.args(), status=status), want, w, kind)
    assert int(status) == 0


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g3", "g16"])
@pytest.mark.parametrize("seqs", [[64, 1], [65], [7] * 20, [0, 33, 0, 0, 2], [129, 63, 64]])
def test_group_sizes(cuda, kind, layout, seqs):
    """Groups of a tile's rows, one more, many small ones, empty ones."""
    n = sum(seqs)
    b = Batch([(i * 97) % 300 for i in range(len(seqs))], seqs, [(i * 13) % 40 for i in range(n)], 16, layout, kind, 15)
    check(B.flash_attn_paged_shared(*b.args()), *b.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
def test_many_heads_share_keys(cuda, kind):
    """More query heads a KV head than a tile has rows."""
    g = torch.Generator(device="cuda").manual_seed(17)
    b = Batch([150], [3], [20, 0, 5], 16, "g20", kind, 17)
    b.q = torch.randn((3, 150, 64), device=cuda, generator=g).to(DT[kind])
    check(B.flash_attn_paged_shared(*b.args()), *b.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
def test_wide_tables(cuda, kind):
    """Tables far wider than the prefixes in them (F32: too wide for planes, so F32 arithmetic)."""
    b = many("g2", kind, 19)
    wide = torch.full((2, 200000 if kind == "f32" else 3000), -1, dtype=torch.int32, device=cuda)
    wide[:, :b.prefix_table.shape[1]] = b.prefix_table
    b.prefix_table = wide
    check(B.flash_attn_paged_shared(*b.args()), *b.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
def test_in_a_graph(cuda, kind):
    b = many("g2", kind, 21)
    a = [t.clone() for t in b.args()]
    B.flash_attn_paged_shared(*a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = B.flash_attn_paged_shared(*a)
    for lens in ([700, 130], [1, 0], [128, 129]):
        b.prefix = lens
        a[4].copy_(ints(lens))
        a[0].copy_(a[0].flip(0))
        b.q = a[0]
        for _ in range(2):
            graph.replay()
        check(out, *b.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g2d64", "g16"])
def test_long_and_short_own_keys_beside_prefixes(cuda, kind, layout):
    """Any split of the work between the prefixes' kernel and the own keys', whose shares depend on the lengths alone."""
    full = [(i * 389) % 2500 for i in range(48)]
    b = Batch([8000, 300], [37, 9], full, 16, layout, kind, 23)
    a = list(b.args())
    for prefix in ([8000, 300], [1000, 300], [1, 0], [0, 129]):
        for own in (full, [0] * 48, [min(n, 1) for n in full], [min(n, 130) for n in full], [n if i % 16 == 5 else 0 for i, n in enumerate(full)]):
            b.prefix, b.own = prefix, own
            a[4], a[7] = ints(prefix), ints(own)
            check(B.flash_attn_paged_shared(*a), *b.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g1", "g2", "g2d64", "g4", "g16"])
@pytest.mark.parametrize("wide", [False, True])
def test_few_sequences(cuda, kind, layout, wide):
    """One launch, with the prefixes' keys as the sequences' first or (tables wider than 4096 positions) as parts."""
    b = Batch([301, 0, 47], [2, 1, 0], [3, 0, 40, 17][:4 if layout in ("g2d64", "g16") else 3], 16, layout, kind, 25)
    b.group.pop(3, None)
    if wide:
        table = torch.full((3, 400), -1, dtype=torch.int32, device=cuda)
        table[:, :b.prefix_table.shape[1]] = b.prefix_table
        b.prefix_table = table
    status = ints([0])
    want, w = b.want()
    check(B.flash_attn_paged_shared(*b.args(), status=status), want, w, kind)
    assert int(status) == 0
    used = torch.zeros(b.k.shape[:2], dtype=torch.bool, device=cuda)  # hidden content does not count
    for t, lens in ((b.prefix_table, b.prefix), (b.table, b.own)):
        for i, n in enumerate(lens):
            pos = torch.arange(n, device=cuda)
            used[t[i].long()[pos // 16], pos % 16] = True
    b.k[~used], b.v[~used] = math.nan, math.inf
    check(B.flash_attn_paged_shared(*b.args()), want, w, kind)
    for at in (0, 18):  # a bad block of a prefix clears its group
        keep = int(b.prefix_table[0, at])
        b.prefix_table[0, at] = b.k.shape[0]
        status.zero_()
        got = B.flash_attn_paged_shared(*b.args(), status=status)
        assert int(status) == BAD_POSITION and (got[:2] == 0).all()
        check(got[2:], want[2:], w[2:], kind)
        b.prefix_table[0, at] = keep
    for prefix, cu in (([301, -4, 47], None), ([301, 0, 47], [0, 2, 1, 3])):  # lengths and offsets out of range are reported
        a = list(b.args())
        a[4] = ints(prefix)
        if cu:
            a[5] = ints(cu)
        status.zero_()
        got = B.flash_attn_paged_shared(*a, status=status)
        assert int(status) == BAD_POSITION and torch.isfinite(got.double()).all()
        check(got[:1], want[:1], w[:1], kind)
    b.v[b.prefix_table[0, 2], 5, 0, 9] = math.inf
    rep = b.q.shape[1] // b.k.shape[2]
    got = B.flash_attn_paged_shared(*b.args())
    assert (got[:2, :rep, 9] == math.inf).all() and int((~torch.isfinite(got)).sum()) == 2 * rep


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g2d64", "g4"])
@pytest.mark.parametrize("order", ["tokens", "heads", "apart"])
@pytest.mark.parametrize("block", [8, 16, 24, 256])
def test_pools_in_any_order(cuda, kind, layout, order, block):
    """Pools that lie token by token, head by head, or with room between heads."""
    b = many(layout, kind, 27, block)
    want = b.want()
    n, _, Hkv, D = b.k.shape
    for name in ("k", "v"):
        x = getattr(b, name)
        if order == "heads":
            x = x.transpose(1, 2).contiguous().transpose(1, 2)
        elif order == "apart":
            wide = torch.full((n, block, Hkv, 2 * D), math.nan, dtype=x.dtype, device=cuda)
            wide[..., :D] = x
            x = wide[..., :D]
        setattr(b, name, x)
    check(B.flash_attn_paged_shared(*b.args()), *want, kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout,n", [("g16", 48), ("g4", 200), ("g20", 30), ("g16", 30)])
def test_groups_that_overlap(cuda, kind, layout, n):
    """Offsets out of order that make groups overlap are reported; whatever such a row shows is no old content."""
    b = Batch([500, 60, 300, 60, 700], [n], [(i * 7) % 40 for i in range(n)], 16, layout, kind, 29)
    a = list(b.args())
    end = n - 1
    a[5] = ints([0, end, 0, end, 0, end])
    groups = b.keys(0)[0].shape[0] - b.own[0]
    assert groups == 500
    status = ints([0])
    seen = []
    for fill in (0xFF, 0x00, 0x7F):
        ws = torch.full((1 << 27,), fill, dtype=torch.uint8, device=cuda)
        status.zero_()
        seen.append(B.flash_attn_paged_shared(*a, workspace=ws, status=status))
        assert int(status) == BAD_POSITION
        assert torch.isfinite(seen[-1].double()).all()
    alone = B.flash_attn_paged_batch(b.q[end:].contiguous(), b.k, b.v, b.table[end:].contiguous(), ints(b.own[end:]))
    for got in seen:
        assert torch.allclose(got[end:].double(), alone.double(), rtol=1e-2, atol=1e-2)
