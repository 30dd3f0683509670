"""The 8-bit paged cache (b200_paged_kv_append_q8, b200_paged_kv_read_q8, b200_flash_attn_paged_batch_q8).

What is held and what is read back is compared exactly with the definition in float64: the scale is a power of two, so an
element is rounded once. Attention is compared with the formula in float64 over the values that the cache stands for;
bounds per output element with `want` exact: the output's one rounding u |want| (u = 2^-11 / 2^-8 for F16 / BF16, half
their epsilon), and 1e-5 of |want| + RMS(want), the bar of the F32 kernels (test_gpu_ops.py), for all else: Q rows and
weights enter as 22 bits, sums are F32; 2^-25 for F16 outputs below its normals.
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
           "g7": (7, 1, 64), "g16": (16, 1, 128), "g20": (20, 1, 64), "g9": (18, 2, 128)}
BAD_POSITION = 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def cumulative(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device="cuda")


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def held(x):
    """The definition in float64: elements as numbers, scales as exponents (255: NaN) of rows x (..., D)."""
    x = x.double()
    top = x.abs().amax(-1)
    odd = ~torch.isfinite(x).all(-1)
    m, e = torch.frexp(torch.where(odd, torch.zeros_like(top), top))
    e = torch.where(m > 0.875, e - 8, e - 9)
    e = torch.where(odd | (top == 0), torch.full_like(e, -127), e).clamp(min=-127)
    y = torch.where(odd[..., None], torch.zeros_like(x), x) * torch.exp2(-e.double())[..., None]
    _, place = torch.frexp(y.abs().clamp(min=2.0 ** -6))  # y in [2^(place - 1), 2^place)
    step = torch.exp2(place.double() - 4.0)
    q = torch.round(y / step) * step  # ties to even
    return q, torch.where(odd, torch.full_like(e, 255), e + 127).to(torch.uint8)


class Cache:
    """A pool in random order with other content in it, and the tables of sequences of given lengths."""

    def __init__(self, lens, block, Hkv, D, seed, spare=3):
        g = gen(seed)
        per = [-(-n // block) for n in lens]
        n = sum(per) + spare
        self.block, self.Hkv, self.D = block, Hkv, D
        self.k = torch.randint(0, 127, (n, block, Hkv, D), device="cuda", generator=g).to(torch.uint8).view(torch.float8_e4m3fn)
        self.v = torch.randint(0, 127, (n, block, Hkv, D), device="cuda", generator=g).to(torch.uint8).view(torch.float8_e4m3fn)
        self.ks = torch.randint(120, 130, (n, Hkv, block), device="cuda", generator=g).to(torch.uint8).view(torch.float8_e8m0fnu)
        self.vs = torch.randint(120, 130, (n, Hkv, block), device="cuda", generator=g).to(torch.uint8).view(torch.float8_e8m0fnu)
        order = torch.randperm(n, device="cuda", generator=g).to(torch.int32)
        self.table = torch.full((len(lens), max(1, max(per))), -5, dtype=torch.int32, device="cuda")  # (unused entries name no block)
        at = 0
        for i, c in enumerate(per):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.lens = list(lens)
        self.seq_lens = ints(lens)

    @property
    def args(self):
        return self.k, self.v, self.ks, self.vs

    def bytes(self):
        return [t.view(torch.uint8).clone() for t in self.args]

    def fill(self, k, v, cu, status=None):
        B.paged_kv_append_q8(k, v, cu, self.seq_lens, *self.args, self.table, status=status)

    def places(self, s, first, last):
        pos = torch.arange(first, last, device="cuda")
        return self.table[s].long()[pos // self.block], pos % self.block

    def values(self, s):
        """The values of sequence s in float64, (len, Hkv, D) each."""
        page, place = self.places(s, 0, self.lens[s])
        out = []
        for q, e in ((self.k, self.ks), (self.v, self.vs)):
            x = q.view(torch.uint8)[page, place].view(torch.float8_e4m3fn).double()
            out.append(x * e.view(torch.uint8)[page, :, place].view(torch.float8_e8m0fnu).double()[..., None])
        return out


def expect_appended(c, before, k, v, new):
    """What the cache's bytes have to be after the append of packed rows k, v."""
    at = 0
    for s, n in enumerate(new):
        page, place = c.places(s, c.lens[s] - n, c.lens[s])
        for rows, q, e in ((k, 0, 2), (v, 1, 3)):
            y, b = held(rows[at:at + n])
            before[q][page, place] = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
            before[e][page, :, place] = b
        at += n
    return before


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("heads", [(8, 128), (4, 64), (1, 128), (3, 64), (1, 64), (20, 128)])
@pytest.mark.parametrize("block,new,past", [(16, [1], [0]), (16, [1, 1, 1], [0, 15, 300]), (7, [37, 0, 5], [0, 9, 13]),
                                            (100, [129, 3], [77, 0]), (1, [4, 2], [0, 3])])
def test_append_holds_the_definition(cuda, kind, heads, block, new, past):
    Hkv, D = heads
    g = gen(block + len(new))
    c = Cache([a + b for a, b in zip(new, past)], block, Hkv, D, 3)
    rows = [(torch.randn((sum(new), Hkv, D), device=cuda, generator=g)
             * torch.exp2(torch.randint(-9, 9, (sum(new), Hkv, 1), device=cuda, generator=g).float())).to(DT[kind]) for _ in range(2)]
    before = c.bytes()
    c.fill(*rows, cumulative(new))
    for got, want in zip(c.bytes(), expect_appended(c, before, *rows, new)):
        # (a zero's sign follows the element's)
        assert torch.equal(got, want)


def test_append_values_at_borders(cuda):
    """Zeros, subnormals, the largest number, ties, the border between two scales, and rows that are no numbers."""
    D = 64
    tiny = 2.0 ** -149
    tops = [0.0, tiny, 2.0 ** -126, 448.0, float(np.nextafter(np.float32(448), np.float32(500))), 1.0, 3.4028234663852886e38,
            2.0 ** -120, 240.0]
    x = torch.zeros((len(tops) + 4, 1, D), device=cuda)
    for i, t in enumerate(tops):
        x[i, 0, 0] = t
        x[i, 0, 1] = -t
        x[i, 0, 2:30] = torch.arange(28, device=cuda) * (t / 27 if t < 1e38 else 1e37)
        x[i, 0, 30] = t * 2.0 ** -18  # below the least step
        x[i, 0, 31] = -0.0
    n = len(tops)
    x[n, 0, :48] = torch.arange(48, device=cuda) * 0.5 + 16.5  # ties between neighbours
    x[n, 0, 60] = 448
    x[n + 1, 0, 5] = math.inf
    x[n + 2, 0, 6] = math.nan
    x[n + 3, 0, 7] = -math.inf
    c = Cache([len(x)], 16, 1, D, 5)
    before = c.bytes()
    c.fill(x, x, cumulative([len(x)]))
    want = expect_appended(c, before, x, x, [len(x)])
    for got, w in zip(c.bytes(), want):
        assert torch.equal(got, w)
    k, v = c.values(0)
    assert torch.isnan(k[n + 1:]).all() and torch.isfinite(k[:n + 1]).all()
    # each element within half a step: 2^-4 of it, or 2^-10 of its row's scale
    _, e = held(x[:n + 1])
    bound = torch.maximum(2.0 ** -4 * x[:n + 1].double().abs(), torch.exp2(e.double() - 137)[..., None])
    assert ((k[:n + 1] - x[:n + 1].double()).abs() <= bound).all()


def test_append_half_types_at_borders(cuda):
    for kind, most in (("f16", 65504.0), ("bf16", 3.3895313892515355e38)):
        x = torch.zeros((4, 2, 128), device=cuda, dtype=DT[kind])
        x[0, 0, 3], x[0, 1, 4], x[1, 0, 5] = most, -most, math.inf
        x[1, 1, 6], x[2, 0, :] = math.nan, 2.0 ** -24 if kind == "f16" else 2.0 ** -133
        x[3] = torch.arange(256, device=cuda).view(2, 128).to(DT[kind])
        c = Cache([4], 2, 2, 128, 6)
        before = c.bytes()
        c.fill(x, x, cumulative([4]))
        for got, w in zip(c.bytes(), expect_appended(c, before, x, x, [4])):
            assert torch.equal(got, w)


def test_append_strided_rows_and_scales(cuda):
    """Rows inside a projection's output, a pool inside a wider tensor, scales with the head axis innermost."""
    g = gen(2)
    wide = torch.randn((9, 12, 128), device=cuda, generator=g).to(torch.bfloat16)
    k, v = wide[:, 4:8], wide[:, 8:]
    c = Cache([9], 4, 4, 128, 8)
    pools = [torch.zeros((6, 4, 6, 160), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn)[:, :, 1:5, 16:144] for _ in range(2)]
    scales = [torch.zeros((6, 4, 4), dtype=torch.uint8, device=cuda).view(torch.float8_e8m0fnu).transpose(1, 2) for _ in range(2)]
    cu = cumulative([9])
    c.fill(k, v, cu)
    B.paged_kv_append_q8(k, v, cu, c.seq_lens, *pools, *scales, c.table)
    page, place = c.places(0, 0, 9)
    for a, b in zip((c.k, c.v), pools):
        assert torch.equal(a.view(torch.uint8)[page, place], b.view(torch.uint8)[page, place])
    for a, b in zip((c.ks, c.vs), scales):
        assert torch.equal(a.view(torch.uint8)[page, :, place], b.view(torch.uint8)[page, :, place])
    out = [torch.zeros((9, 6, 128), device=cuda)[:, 1:5] for _ in range(2)]
    got = B.paged_kv_read_q8(cu, c.seq_lens, 9, *pools, *scales, c.table, k=out[0], v=out[1])
    for x, y in zip(got, c.values(0)):
        assert torch.equal(x.double(), y)


def test_append_bad_offsets_and_blocks(cuda):
    """What names no place is skipped and reported; everything else is written."""
    g = gen(4)
    c = Cache([20, 30], 8, 2, 64, 9)
    k = torch.randn((12, 2, 64), device=cuda, generator=g)
    good = c.bytes()
    status = ints([0])
    c.table[0, 2] = 99  # positions 16 .. 19 of the first sequence
    B.paged_kv_append_q8(k, k, ints([0, 6, 12]), c.seq_lens, *c.args, c.table, status=status)
    want = [t.clone() for t in good]
    for s, rows, first in ((0, k[:2], 14), (1, k[6:], 24)):
        page, place = c.places(s, first, first + len(rows))
        y, b = held(rows)
        for q, e in ((0, 2), (1, 3)):
            want[q][page, place] = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
            want[e][page, :, place] = b
    assert int(status) == BAD_POSITION
    for got, w in zip(c.bytes(), want):
        assert torch.equal(got, w)
    status.zero_()
    B.paged_kv_append_q8(k, k, ints([0, 6, 12]), ints([3, 1000]), *c.args, c.table, status=status)  # before 0, past the table
    assert int(status) == BAD_POSITION
    page, place = c.places(0, 0, 3)
    y, b = held(k[3:6])
    want[0][page, place] = want[1][page, place] = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
    want[2][page, :, place] = want[3][page, :, place] = b
    for got, w in zip(c.bytes(), want):
        assert torch.equal(got, w)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("heads", [(8, 128), (3, 64), (1, 64), (20, 128)])
@pytest.mark.parametrize("block,lens,rows", [(16, [1], [1]), (16, [300, 0, 33], [300, 0, 33]), (7, [40, 90], [3, 90]),
                                             (128, [129, 700, 5], [100, 700, 0])])
def test_read(cuda, kind, heads, block, lens, rows):
    c = Cache(lens, block, *heads, 11)
    got = B.paged_kv_read_q8(cumulative(rows), c.seq_lens, sum(rows), *c.args, c.table, dtype=DT[kind])
    for which in range(2):
        want = torch.cat([c.values(s)[which][lens[s] - rows[s]:] for s in range(len(lens))])
        assert got[which].dtype == DT[kind] and torch.equal(got[which], want.to(DT[kind]))


def test_read_values(cuda):
    """Scales at both ends, NaN among them, all elements; F16 rounds and overflows as a conversion does."""
    c = Cache([255], 16, 4, 64, 12)
    every = torch.arange(256, device=cuda).to(torch.uint8).view(1, 1, 4, 64)
    c.k.view(torch.uint8).copy_(every)
    c.v.view(torch.uint8).copy_(every.flip(-1))
    n = torch.arange(c.ks.numel(), device=cuda)
    c.ks.view(torch.uint8).copy_((n % 256).to(torch.uint8).view(c.ks.shape))
    c.vs.view(torch.uint8).copy_((255 - n % 256).to(torch.uint8).view(c.ks.shape))
    for kind in DT:
        got = B.paged_kv_read_q8(cumulative([255]), c.seq_lens, 255, *c.args, c.table, dtype=DT[kind])
        for x, want in zip(got, c.values(0)):
            want = want.float().to(DT[kind])  # (exact in F32 but beyond its largest)
            assert torch.equal(torch.isnan(x), torch.isnan(want))
            assert torch.equal(torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf),
                               torch.nan_to_num(want, nan=0.0, posinf=math.inf, neginf=-math.inf))


def test_read_outside_and_bad(cuda):
    """Rows outside every sequence stay; rows whose position, block or offsets are out of range are zero, and reported."""
    c = Cache([20, 30], 8, 2, 64, 13)
    k, v = torch.full((40, 2, 64), 7.0, device=cuda), torch.full((40, 2, 64), 7.0, device=cuda)
    status = ints([0])
    B.paged_kv_read_q8(ints([5, 25, 30]), c.seq_lens, 40, *c.args, c.table, k=k, v=v, status=status)
    assert int(status) == 0
    for t, which in ((k, 0), (v, 1)):
        assert (t[:5] == 7).all() and (t[30:] == 7).all()
        assert torch.equal(t[5:25].double(), c.values(0)[which]) and torch.equal(t[25:30].double(), c.values(1)[which][25:])
    good = c.values(1)
    c.table[0, 1] = -1
    k, v = B.paged_kv_read_q8(ints([0, 20, 50]), c.seq_lens, 50, *c.args, c.table, dtype=torch.float32, status=status)
    assert int(status) == BAD_POSITION
    assert (k[8:16] == 0).all() and (v[8:16] == 0).all() and torch.equal(k[20:].double(), good[0])
    status.zero_()
    k, v = B.paged_kv_read_q8(ints([0, 10, 30]), ints([4, 30]), 30, *c.args, c.table, dtype=torch.float32, status=status)
    assert int(status) == BAD_POSITION and (k[:6] == 0).all() and torch.equal(k[10:].double(), good[0][10:])
    status.zero_()
    k, v = torch.full((30, 2, 64), 7.0, device=cuda), torch.full((30, 2, 64), 7.0, device=cuda)
    B.paged_kv_read_q8(ints([0, 10, 40]), c.seq_lens, 30, *c.args, c.table, k=k, v=v, status=status)  # 40 > 30
    assert int(status) == BAD_POSITION and (k[10:] == 0).all()


def exact(q, k, v, scale=None):
    """One query row (Hq, D) over k, v (m, Hkv, D), float64."""
    Hq, D = q.shape
    if k.shape[0] == 0:
        return torch.zeros((Hq, D), dtype=torch.float64, device=q.device)
    rep = Hq // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    s = torch.einsum("hd,mhd->hm", q.double(), k) * (scale or 1 / math.sqrt(D))
    return torch.einsum("hm,mhd->hd", torch.softmax(s, -1), v)


def check(got, want, kind, rms=None):
    assert torch.isfinite(got.double()).all()
    rms = float(want.square().mean().sqrt()) if rms is None else rms
    bound = UNIT[kind] * want.abs() + 1e-5 * (want.abs() + rms) + (2.0 ** -25 if kind == "f16" else 0.0)
    worst = float(((got.double() - want).abs() / bound.clamp(min=1e-300)).max()) if got.numel() else 0.0
    assert worst <= 1.0, worst


def filled(lens, block, Hkv, D, seed, kind="f32", key=1.0):
    c = Cache(lens, block, Hkv, D, seed)
    g = gen(seed + 1)
    k = (torch.randn((sum(lens), Hkv, D), device="cuda", generator=g) * key).to(DT[kind])
    v = (torch.randn((sum(lens), Hkv, D), device="cuda", generator=g) + 0.5).to(DT[kind])
    c.fill(k, v, cumulative(lens))
    return c


def decode_want(c, q, scale=None):
    return torch.stack([exact(q[s], *c.values(s), scale) for s in range(len(c.lens))])


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("block,lens", [(16, [1]), (16, [301]), (8, [5, 0, 1, 64, 33, 129, 1000]), (100, [77, 2500, 0, 100]),
                                        (1, [40, 3]), (5000, [4999, 2])],
                         ids=["single", "one", "ragged", "pages_of_100", "pages_of_one", "one_page"])
def test_decode(cuda, kind, layout, block, lens):
    Hq, Hkv, D = LAYOUTS[layout]
    c = filled(lens, block, Hkv, D, 21, kind)
    q = torch.randn((len(lens), Hq, D), device=cuda, generator=gen(22)).to(DT[kind])
    check(B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens), decode_want(c, q), kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64", "g16", "g9"])
def test_decode_many_and_long(cuda, kind, layout):
    Hq, Hkv, D = LAYOUTS[layout]
    lens = [(i * 1277) % 4090 + 1 for i in range(40)] + [9001, 0, 0, 17]
    c = filled(lens, 32, Hkv, D, 31, kind)
    q = torch.randn((len(lens), Hq, D), device=cuda, generator=gen(32)).to(DT[kind])
    want = decode_want(c, q)
    got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens)
    check(got, want, kind)
    n = B.lib().b200_flash_attn_paged_batch_q8_workspace_bytes(len(lens), c.table.shape[1] * 32, D, Hq, Hkv)
    for fill in (0, 0x7C, 0xFF):  # what a workspace held before is never read
        ws = torch.full((n,), fill, dtype=torch.uint8, device=cuda)
        assert torch.equal(B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens, workspace=ws), got)


@pytest.mark.parametrize("kind", list(DT))
def test_decode_strides_and_scale(cuda, kind):
    lens = [50, 700, 3]
    c = filled(lens, 16, 2, 128, 41, kind)
    wide = torch.randn((3, 9, 160), device=cuda, generator=gen(42)).to(DT[kind])
    q, out = wide[:, 1:7, 16:144], torch.zeros((3, 8, 128), device=cuda, dtype=DT[kind])
    got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens, scale=0.3, out=out[:, 2:])
    check(got, decode_want(c, q, 0.3), kind)
    assert (out[:, :2] == 0).all()


@pytest.mark.parametrize("layout", ["g2", "g2d64", "g16"])
def test_decode_growing_scores_and_spread_magnitudes(cuda, layout):
    """Scores that grow along the keys, V rows whose scales differ by up to 2^60, Q rows far from 1."""
    Hq, Hkv, D = LAYOUTS[layout]
    n = 900
    g = gen(51)
    c = Cache([n, n, n], 16, Hkv, D, 50)
    k = torch.randn((3 * n, Hkv, D), device=cuda, generator=g) * torch.linspace(0.1, 4.0, n, device=cuda).repeat(3)[:, None, None]
    v = torch.randn((3 * n, Hkv, D), device=cuda, generator=g)
    v[n:2 * n] *= torch.exp2(torch.randint(-30, 31, (n, Hkv, 1), device=cuda, generator=g).float())
    k[2 * n:] *= 2.0 ** 60
    c.fill(k, v, cumulative([n] * 3))
    q = torch.randn((3, Hq, D), device=cuda, generator=g)
    q[2] *= 2.0 ** -60
    got, want = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens), decode_want(c, q)
    for s in range(3):
        check(got[s], want[s], "f32")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["g2", "g2d64", "g16"])
@pytest.mark.parametrize("up", [105, -105])
def test_decode_large_rows_of_q_with_small_keys(cuda, kind, layout, up):
    """Rows of Q and keys at the two ends of the exponents' range, whose products lie in its middle."""
    Hq, Hkv, D = LAYOUTS[layout]
    g = gen(60)
    c = Cache([300, 17], 16, Hkv, D, 61)
    k, v = (torch.randn((317, Hkv, D), device=cuda, generator=g) for _ in range(2))
    c.fill(k * 2.0 ** -up, v, cumulative(c.lens))
    q = (torch.randn((2, Hq, D), device=cuda, generator=g) * 2.0 ** up).to(DT[kind])
    check(B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens), decode_want(c, q), kind)


def test_decode_light_keys_with_large_values(cuda):
    """A key whose weight is 2^-40 of the heaviest and whose V row is 2^50 of the others' decides the output."""
    n, D = 64, 128
    g = gen(53)
    c = Cache([n], 16, 1, D, 52)
    k = torch.zeros((n, 1, D), device=cuda)
    k[:, 0, 0] = 40.0 * math.log(2.0)
    k[5, 0, 0] = 0.0
    v = torch.randn((n, 1, D), device=cuda, generator=g)
    v[5] *= 2.0 ** 50
    c.fill(k, v, cumulative([n]))
    q = torch.zeros((1, 2, D), device=cuda)
    q[0, 0, 0], q[0, 1, 0] = 1.0, 0.5
    check(B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens, scale=1.0), decode_want(c, q, 1.0), "f32")


@pytest.mark.parametrize("kind", list(DT))
def test_decode_nan_and_hidden_bytes(cuda, kind):
    """Scales of NaN reach the rows that see them; whatever lies behind a sequence's end, in its last block and in unused
    blocks, does not. Elements of NaN (127) count as NaN."""
    lens = [40, 90, 3, 0]
    c = filled(lens, 16, 2, 128, 61, kind)
    q = torch.randn((4, 8, 128), device=cuda, generator=gen(62)).to(DT[kind])
    want = decode_want(c, q)
    used = torch.zeros((c.k.shape[0], 16), dtype=torch.bool, device=cuda)
    for s in range(4):
        used[c.places(s, 0, lens[s])] = True
    for t in (c.k, c.v):
        t.view(torch.uint8)[~used] = 127
    for t in (c.ks, c.vs):
        t.view(torch.uint8).transpose(1, 2)[~used] = 255
    check(B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens), want, kind)
    page, place = c.places(0, 39, 40)
    c.ks.view(torch.uint8)[page, 0, place] = 255
    page, place = c.places(1, 0, 1)
    c.vs.view(torch.uint8)[page, 1, place] = 255
    page, place = c.places(2, 1, 2)
    c.v.view(torch.uint8)[page, place, 0, 9] = 127
    got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens)
    assert torch.isnan(got[0, :4]).all() and torch.isnan(got[1, 4:]).all()
    assert torch.isnan(got[2, :4, 9]).all() and int(torch.isnan(got[2]).sum()) == 4
    rms = float(want.square().mean().sqrt())
    check(got[0, 4:], want[0, 4:], kind, rms)
    check(got[1, :4], want[1, :4], kind, rms)
    check(got[2, 4:], want[2, 4:], kind, rms)
    assert (got[3] == 0).all()
    q[1, 2] = math.nan
    got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens)
    assert torch.isnan(got[1, 2]).all() and torch.isfinite(got[1, :2]).all()


def test_decode_bad_blocks_and_lengths(cuda):
    """Keys in blocks out of range are left out, lengths are cut to the table, and both are reported."""
    lens = [40, 90]
    c = filled(lens, 16, 2, 64, 71)
    q = torch.randn((2, 4, 64), device=cuda, generator=gen(72))
    status = ints([0])
    k, v = c.values(1)
    c.table[1, 2] = 1000
    keep = torch.ones(90, dtype=torch.bool, device=cuda)
    keep[32:48] = False
    got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens, status=status)
    assert int(status) == BAD_POSITION
    check(got[1], exact(q[1], k[keep], v[keep]), "f32")
    check(got[0], exact(q[0], *c.values(0)), "f32")
    for lens2 in ([-3, 90], [-2 ** 31, 90]):
        status.zero_()
        got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, ints(lens2), status=status)
        assert int(status) == BAD_POSITION and (got[0] == 0).all()
        check(got[1], exact(q[1], k[keep], v[keep]), "f32")
    full = filled([96, 96], 16, 2, 64, 73)
    status.zero_()
    got = B.flash_attn_paged_batch_q8(q, *full.args, full.table, ints([2 ** 31 - 1, 97]), status=status)
    assert int(status) == BAD_POSITION
    check(got, decode_want(full, q), "f32")
    full.table.fill_(-1)  # no key is left
    assert (B.flash_attn_paged_batch_q8(q, *full.args, full.table, full.seq_lens) == 0).all()


def test_decode_offsets_past_32_bits(cuda):
    """Blocks that lie more than 2^31 and 2^32 bytes into the pool."""
    Hkv, D, block = 8, 128, 256
    n = 2 ** 32 // (block * Hkv * D) + 5
    pools = [torch.empty((n, block, Hkv, D), dtype=torch.uint8, device=cuda).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.empty((n, Hkv, block), dtype=torch.uint8, device=cuda).view(torch.float8_e8m0fnu) for _ in range(2)]
    table = ints([[n - 1, n // 2, 0]])
    g = gen(81)
    k, v = (torch.randn((700, Hkv, D), device=cuda, generator=g) for _ in range(2))
    B.paged_kv_append_q8(k, v, cumulative([700]), ints([700]), *pools, *scales, table)
    got = B.paged_kv_read_q8(cumulative([700]), ints([700]), 700, *pools, *scales, table, dtype=torch.float32)
    for x, rows in zip(got, (k, v)):
        y, e = held(rows)
        assert torch.equal(x.double(), y * torch.exp2(e.double() - 127)[..., None])
    q = torch.randn((1, 16, D), device=cuda, generator=g)
    check(B.flash_attn_paged_batch_q8(q, *pools, *scales, table, ints([700])), exact(q[0], *(x.double() for x in got))[None], "f32")


def test_empty_calls(cuda):
    c = Cache([5], 4, 2, 64, 91)
    e = torch.zeros((0, 2, 64), device=cuda)
    B.paged_kv_append_q8(e, e, ints([0, 0]), ints([0]), *c.args, c.table)
    k, v = B.paged_kv_read_q8(ints([0, 0]), ints([0]), 0, *c.args, c.table)
    assert k.shape == (0, 2, 64)
    assert B.flash_attn_paged_batch_q8(torch.zeros((0, 4, 64), device=cuda), *c.args, c.table[:0], ints([])).shape == (0, 4, 64)


def test_argument_errors(cuda):
    c = Cache([5], 4, 2, 64, 92)
    k = torch.zeros((5, 2, 64), device=cuda)
    cu = cumulative([5])
    for bad in (lambda: B.paged_kv_append_q8(k, k[:4], cu, c.seq_lens, *c.args, c.table),
                lambda: B.paged_kv_append_q8(k, k.half(), cu, c.seq_lens, *c.args, c.table),
                lambda: B.paged_kv_append_q8(k, k, cu, c.seq_lens, c.k, c.v, c.ks[:1], c.vs[:1], c.table),
                lambda: B.paged_kv_append_q8(k, k, cu, c.seq_lens, c.k.view(torch.uint8), c.v, c.ks, c.vs, c.table),
                lambda: B.paged_kv_append_q8(k, k, cu, c.seq_lens, c.k, c.v, c.ks.view(torch.uint8), c.vs, c.table),
                lambda: B.paged_kv_append_q8(k.cpu(), k, cu, c.seq_lens, *c.args, c.table),
                lambda: B.paged_kv_read_q8(cu, c.seq_lens, 5, *c.args, c.table, k=k),
                lambda: B.paged_kv_read_q8(cu, c.seq_lens, 4, *c.args, c.table, k=k, v=k.clone()),
                lambda: B.flash_attn_paged_batch_q8(k[:1, :1].double(), *c.args, c.table, c.seq_lens),
                lambda: B.flash_attn_paged_batch_q8(torch.zeros((1, 3, 64), device=cuda), *c.args, c.table, c.seq_lens)):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(B.B200Error):
        B.paged_kv_append_q8(torch.zeros((5, 2, 72), device=cuda)[..., 2:66], k, cu, c.seq_lens, *c.args, c.table)
