"""b200_flash_attn_paged_shared against the formula in float64.

Bounds as for the packed attention (test_gpu_batch.py): per output element with `want` exact, the output's one rounding
u |want| (u = 2^-11 / 2^-8 for F16 / BF16, half their epsilon); a prefix's weights are rounded to the type before the
second product, so its terms p_j v_j move by at most u each, independently: a standard deviation of at most u / sqrt(3)
of W = sqrt(sum (p_j v_j)^2), allowed 4 u W (seven deviations); 1e-5 of |want| + RMS(want) for the rest; 2^-25 for F16
outputs below its normals.
"""
import math

import pytest
import torch

import b200infer as B

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LAYOUTS = {"g2": (16, 8, 128), "g4": (32, 8, 128), "g2d64": (8, 4, 64), "g1": (3, 3, 64), "g3": (6, 2, 128),
           "g7": (7, 1, 64), "g16": (16, 1, 128), "g20": (20, 1, 64)}
BAD_POSITION = 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Batch:
    """Groups of sequences behind prefixes, over one pool in random order. seqs: sequences of each group."""

    def __init__(self, prefix, seqs, lens, block, layout, kind, seed, first=0):
        Hq, Hkv, D = LAYOUTS[layout]
        g = gen(seed)
        per = [-(-n // block) for n in list(prefix) + list(lens)]
        n = sum(per) + 3
        self.block, self.prefix, self.seqs, self.own, self.kind = block, list(prefix), list(seqs), list(lens), kind
        self.k = torch.randn((n, block, Hkv, D), device="cuda", generator=g).to(DT[kind])
        self.v = (torch.randn((n, block, Hkv, D), device="cuda", generator=g) + 0.5).to(DT[kind])
        self.q = torch.randn((len(lens), Hq, D), device="cuda", generator=g).to(DT[kind])
        order = torch.randperm(n, device="cuda", generator=g).to(torch.int32)
        G = len(prefix)
        self.prefix_table = torch.full((G, max([1] + per[:G])), -7, dtype=torch.int32, device="cuda")
        self.table = torch.full((len(lens), max([1] + per[G:])), -7, dtype=torch.int32, device="cuda")
        at = 0
        for i, c in enumerate(per):
            row = self.prefix_table[i] if i < G else self.table[i - G]
            row[:c] = order[at:at + c]
            at += c
        cu = [first]
        for s in seqs:
            cu.append(cu[-1] + s)
        self.cu = ints(cu)
        self.group = {}
        for i in range(len(seqs)):
            for s in range(cu[i], cu[i + 1]):
                self.group[s] = i

    def args(self):
        return (self.q, self.k, self.v, self.prefix_table, ints(self.prefix), self.cu, self.table, ints(self.own))

    def rows(self, pool, table, n):
        pos = torch.arange(n, device="cuda")
        return pool[table.long()[pos // self.block], pos % self.block]

    def keys(self, s):
        g = self.group.get(s)
        out = []
        for pool in (self.k, self.v):
            head = [] if g is None else [self.rows(pool, self.prefix_table[g], self.prefix[g])]
            out.append(torch.cat(head + [self.rows(pool, self.table[s], self.own[s])]))
        return out

    def want(self, scale=None):
        pairs = [exact(self.q[s], *self.keys(s), scale) for s in range(len(self.own))]
        return torch.stack([a for a, _ in pairs]), torch.stack([b for _, b in pairs])


def exact(q, k, v, scale=None):
    Hq, D = q.shape
    if k.shape[0] == 0:
        z = torch.zeros((Hq, D), dtype=torch.float64, device=q.device)
        return z, z
    rep = Hq // k.shape[1]
    k, v = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    s = torch.einsum("hd,mhd->hm", q.double(), k) * (scale or 1 / math.sqrt(D))
    p = torch.softmax(s, -1)
    return torch.einsum("hm,mhd->hd", p, v), torch.einsum("hm,mhd->hd", p.square(), v.square()).sqrt()


def check(got, want, w, kind):
    assert torch.isfinite(got.double()).all()
    u = UNIT[kind]
    rms = float(want.square().mean().sqrt())
    bound = u * want.abs() + 4 * u * w + 1e-5 * (want.abs() + rms) + (2.0 ** -25 if kind == "f16" else 0.0)
    worst = float(((got.double() - want).abs() / bound.clamp(min=1e-300)).max()) if got.numel() else 0.0
    assert worst <= 1.0, worst


SHAPES = {
    "one": ([1], [1], [1], 16),
    "one_of_each": ([37], [3], [5, 0, 12], 16),
    "groups": ([130, 0, 257, 1], [3, 2, 1, 5], [1, 33, 0, 4, 129, 16, 0, 2, 77, 1, 40], 16),
    "odd_pages": ([301, 77], [4, 3], [3, 40, 17, 90, 0, 5, 1], 7),
    "pages_of_100": ([1000, 128], [20, 1], [(i * 37) % 150 for i in range(21)], 100),
}


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("shape", list(SHAPES))
def test_shared(cuda, kind, layout, shape):
    prefix, seqs, lens, block = SHAPES[shape]
    b = Batch(prefix, seqs, lens, block, layout, kind, 3)
    check(B.flash_attn_paged_shared(*b.args()), *b.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64", "g16"])
def test_long_prefix_many_rows(cuda, kind, layout):
    b = Batch([5003, 700], [61, 9], [(i * 131) % 900 for i in range(70)], 32, layout, kind, 5)
    got = B.flash_attn_paged_shared(*b.args())
    check(got, *b.want(), kind)
    Hq, Hkv, D = LAYOUTS[layout]
    n = B.lib().b200_flash_attn_paged_shared_workspace_bytes(70, b.table.shape[1] * 32, 2, b.prefix_table.shape[1] * 32, D, Hq, Hkv,
                                                             list(DT).index(kind))
    for fill in (0, 0x7C, 0xFF):  # what a workspace held before is never read
        ws = torch.full((n,), fill, dtype=torch.uint8, device=cuda)
        assert torch.equal(B.flash_attn_paged_shared(*b.args(), workspace=ws), got)


@pytest.mark.parametrize("kind", list(DT))
def test_equals_unshared(cuda, kind):
    """Without groups, and with prefixes of no positions, it is the batched decode; sequences outside every group see their
    own positions alone."""
    b = Batch([40, 0], [2, 2], [50, 3, 700, 1, 90, 0, 2], 16, "g4", kind, 7, first=1)  # sequences 0, 5, 6 are in no group
    check(B.flash_attn_paged_shared(*b.args()), *b.want(), kind)
    none = Batch([], [], [50, 3, 700], 16, "g4", kind, 8)
    got = B.flash_attn_paged_shared(*none.args())
    check(got, *none.want(), kind)


@pytest.mark.parametrize("kind", list(DT))
def test_strides_scale_and_growing_scores(cuda, kind):
    b = Batch([300, 20], [3, 4], [50, 3, 70, 1, 90, 0, 2], 16, "g3", kind, 9)
    n = b.k.shape[0]
    wide = torch.zeros((n, 16, 3, 160), device=cuda, dtype=DT[kind])
    pools = [wide[:, :, 1:, 16:144], torch.zeros_like(wide)[:, :, 1:, 16:144]]
    grow = torch.linspace(0.2, 3.0, 16, device=cuda)[None, :, None, None]
    b.k = (b.k.float() * grow).to(DT[kind])
    for t, x in zip(pools, (b.k, b.v)):
        t.copy_(x)
    b.k, b.v = pools
    q = torch.randn((7, 9, 144), device=cuda, generator=gen(10)).to(DT[kind])
    b.q = q[:, 2:8, 8:136]
    out = torch.full((7, 8, 128), 5.0, device=cuda).to(DT[kind])
    got = B.flash_attn_paged_shared(*b.args(), scale=0.2, out=out[:, 1:7])
    check(got, *b.want(0.2), kind)
    assert (out[:, 0] == 5).all() and (out[:, 7] == 5).all()


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g2d64"])
def test_hidden_content(cuda, kind, layout):
    """What lies behind the ends of prefixes and sequences, and in unused blocks, does not count, whatever it is."""
    b = Batch([301, 77, 5], [9, 3, 2], [(i * 29) % 60 for i in range(14)], 16, layout, kind, 11)
    want = b.want()
    used = torch.zeros((b.k.shape[0], 16), dtype=torch.bool, device=cuda)
    for table, lens in ((b.prefix_table, b.prefix), (b.table, b.own)):
        for i, n in enumerate(lens):
            pos = torch.arange(n, device=cuda)
            used[table[i].long()[pos // 16], pos % 16] = True
    for bad in (math.nan, math.inf, -math.inf):
        b.k[~used] = bad
        b.v[~used] = bad
        check(B.flash_attn_paged_shared(*b.args()), *want, kind)


@pytest.mark.parametrize("kind", list(DT))
def test_values_that_are_no_numbers(cuda, kind):
    """A NaN in a key, of the prefix or of a sequence, reaches the rows that see it and no other."""
    b = Batch([200, 90], [3, 2], [20, 0, 5, 7, 30], 16, "g2", kind, 13)
    want, w = b.want()
    b.k[b.prefix_table[0, 3], 4, 2, 5] = math.nan  # heads 4 and 5 of the first group's rows
    b.k[b.table[4, 1], 2, 0, 0] = math.nan         # heads 0 and 1 of the last row
    got = B.flash_attn_paged_shared(*b.args())
    odd = torch.zeros((5, 16), dtype=torch.bool, device=cuda)
    odd[:3, 4:6] = True
    odd[4, :2] = True
    assert torch.isnan(got[odd]).all()
    check(got[~odd], want[~odd], w[~odd], kind)
    # keys whose scores are -inf count for nothing; rows that have only such keys are zero
    b = Batch([40], [2], [3, 0], 16, "g2", kind, 14)
    b.q.fill_(1.0)
    b.k[b.prefix_table[0].long()] = -math.inf
    got = B.flash_attn_paged_shared(*b.args())
    assert (got[1] == 0).all()
    b.prefix = [0]
    want, w = b.want()
    check(got[:1], want[:1], w[:1], kind)


@pytest.mark.parametrize("kind", list(DT))
def test_infinite_values(cuda, kind):
    """An infinite V element that a row sees makes that column of the row infinite."""
    b = Batch([200], [3], [20, 1, 5], 16, "g2d64", kind, 15)
    b.v[b.table[1, 0], 0, 1, 9] = math.inf
    want, w = b.want()
    got = B.flash_attn_paged_shared(*b.args())
    fine = torch.isfinite(want)
    assert torch.equal(got.double()[~fine], want[~fine])
    w = torch.where(fine, w, 0.0)
    check(torch.where(fine, got.double(), 0.0).to(DT[kind]), torch.where(fine, want, 0.0), w, kind)


def test_spread_magnitudes(cuda):
    """F32 rows, columns and keys whose magnitudes differ by far more than one exponent holds."""
    b = Batch([700], [5], [20, 0, 5, 300, 1], 16, "g2", "f32", 17)
    b.v[..., 3] *= 2.0 ** -40
    b.k[b.prefix_table[0, 5]] *= 2.0 ** -30
    b.v[b.prefix_table[0, 6]] *= 2.0 ** 30
    got = B.flash_attn_paged_shared(*b.args())
    want, _ = b.want()
    for d in (3, 4):  # each column by its own magnitude
        rms = float(want[..., d].square().mean().sqrt())
        assert ((got[..., d].double() - want[..., d]).abs() <= 1e-5 * (want[..., d].abs() + rms)).all()


@pytest.mark.parametrize("kind", list(DT))
def test_bad_tables_lengths_and_offsets(cuda, kind):
    b = Batch([200, 90, 64], [3, 2, 1], [20, 0, 5, 7, 30, 3], 16, "g2", kind, 19)
    want, w = b.want()
    status = ints([0])
    got = B.flash_attn_paged_shared(*b.args(), status=status)
    assert int(status) == 0
    check(got, want, w, kind)
    kept = b.prefix_table.clone()
    b.prefix_table[1, 3] = 5000  # the second group's rows are zero
    got = B.flash_attn_paged_shared(*b.args(), status=status)
    assert int(status) == BAD_POSITION and (got[3:5] == 0).all()
    check(got[[0, 1, 2, 5]], want[[0, 1, 2, 5]], w[[0, 1, 2, 5]], kind)
    b.prefix_table.copy_(kept)
    # a sequence's own keys in such a block are left out
    status.zero_()
    kept = b.table.clone()
    b.table[4, 1] = -1
    got = B.flash_attn_paged_shared(*b.args(), status=status)
    assert int(status) == BAD_POSITION
    k, v = (torch.cat([b.rows(x, b.prefix_table[1], 90), b.rows(x, kept[4], 16)]) for x in (b.k, b.v))
    e, f = exact(b.q[4], k, v)
    check(got[4:5], e[None], f[None], kind)
    b.table.copy_(kept)
    # lengths are cut to the table
    for prefix, own in (([2 ** 31 - 1, 90, 64], None), ([-1, 90, 64], None), (None, [20, -7, 5, 7, 30, 3])):
        status.zero_()
        full = Batch([b.prefix_table.shape[1] * 16, 90, 64], [3, 2, 1], [20, 0, 5, 7, 30, 3], 16, "g2", kind, 21)
        a = list(full.args())
        if prefix is not None:
            a[4] = ints(prefix)
            if prefix[0] < 0:
                full.prefix[0] = 0
        if own is not None:
            a[7] = ints(own)
        got = B.flash_attn_paged_shared(*a, status=status)
        assert int(status) == BAD_POSITION
        check(got, *full.want(), kind)
    # offsets out of range: those groups' rows see their own positions alone
    for cu, group in (([0, 3, 2, 6], {0: 0, 1: 0, 2: 2, 3: 2, 4: 2, 5: 2}), ([0, 3, 5, 7], {0: 0, 1: 0, 2: 0, 3: 1, 4: 1})):
        status.zero_()
        b.cu, b.group = ints(cu), group
        got = B.flash_attn_paged_shared(*b.args(), status=status)
        assert int(status) == BAD_POSITION
        check(got[[0, 1, 3, 4, 5]], *(x[[0, 1, 3, 4, 5]] for x in b.want()), kind)


def test_empty_calls_and_argument_errors(cuda):
    b = Batch([20], [2], [3, 4], 16, "g2d64", "f32", 23)
    a = list(b.args())
    z = [a[0][:0], a[1], a[2], a[3], a[4], ints([0, 0]), a[6][:0], a[7][:0]]
    assert B.flash_attn_paged_shared(*z).shape == (0, 8, 64)
    for i, x in ((0, a[0][:, :3]), (1, a[1].half()), (3, a[3].long()), (4, a[4].long()), (5, a[5][:1]), (6, a[6][:1]), (7, a[7].cpu()),
                 (0, a[0].cpu())):
        with pytest.raises((ValueError, TypeError)):
            B.flash_attn_paged_shared(*a[:i], x, *a[i + 1:])
