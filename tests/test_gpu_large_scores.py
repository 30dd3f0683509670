"""Attention with scores far beyond 1: where one key decides, its V row is the answer, however large its score is.

Keys lie along q with factors of which the first or fourth is the largest by 7 % at least: its score is `target`, the others' are
lower by 0.07 target, so by exp(-700) in the weights from 10^4 on, and `want` is that key's V row but for nothing in float64.
The output is that row times 1 as 22 bits give it: bound 1e-5 of |want| plus one rounding u |want|."""
import math

import pytest
import torch

import b200infer as B
from test_gpu_q8 import DT, UNIT, Cache, cumulative, gen, ints

pytestmark = pytest.mark.gpu

TARGETS = [1e4, 3e7, 1e8, 1e10, 1e25]


def rows(n, target, Hq, Hkv, D, kind):
    g = gen(n)
    a = math.sqrt(target * math.sqrt(D))
    q = torch.zeros((Hq, D), device="cuda")
    k = torch.zeros((n, Hkv, D), device="cuda")
    q[:, 0] = a
    k[:, :, 0] = -a * torch.rand((n, Hkv), device="cuda", generator=g)
    k[min(3, n - 1), :, 0] = a
    v = torch.randn((n, Hkv, D), device="cuda", generator=g) * torch.exp2(torch.randint(-3, 4, (n, Hkv, 1), device="cuda", generator=g).float())
    return q.to(DT[kind]), k.to(DT[kind]), v.to(DT[kind])


def possible(kind, target):
    return kind != "f16" or target <= 1e8  # rows of up to 3.4e4


def close(got, want, kind):
    want = want.double().expand_as(got)
    assert torch.isfinite(got.double()).all()
    assert ((got.double() - want).abs() <= (1e-5 + UNIT[kind]) * want.abs()).all()


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", [(16, 8, 128), (8, 4, 64), (16, 1, 128)])
@pytest.mark.parametrize("n", [1, 300])
@pytest.mark.parametrize("seqs", [1, 60])
@pytest.mark.parametrize("target", TARGETS)
def test_8_bit_cache(cuda, kind, layout, n, seqs, target):
    if not possible(kind, target):
        return
    Hq, Hkv, D = layout
    q, k, v = rows(n, target, *layout, kind)
    c = Cache([n], 16, Hkv, D, 3)
    c.fill(k, v, cumulative([n]))
    want = c.values(0)[1][min(3, n - 1)].repeat_interleave(Hq // Hkv, 0)
    got = B.flash_attn_paged_batch_q8(q.expand(seqs, -1, -1).contiguous(), *c.args, c.table.expand(seqs, -1).contiguous(), ints([n] * seqs))
    close(got, want, kind)


@pytest.mark.parametrize("target", [1e4, 1e8, 1e15])
def test_8_bit_cache_equal_scores(cuda, target):
    """Keys of one large score count alike, whatever their V rows' scales are."""
    Hq, Hkv, D = 16, 8, 128
    q, k, _ = rows(1, target, Hq, Hkv, D, "f32")
    v = torch.randn((200, Hkv, D), device=cuda, generator=gen(4)) * torch.exp2(torch.randint(-20, 21, (200, Hkv, 1), device=cuda, generator=gen(5)).float())
    c = Cache([200], 16, Hkv, D, 3)
    c.fill(k.expand(200, -1, -1).contiguous(), v, cumulative([200]))
    want = c.values(0)[1].mean(0).repeat_interleave(2, 0)
    for seqs in (1, 60):
        got = B.flash_attn_paged_batch_q8(q.expand(seqs, -1, -1).contiguous(), *c.args, c.table.expand(seqs, -1).contiguous(),
                                          ints([200] * seqs)).double()
        assert ((got - want).abs() <= 1e-5 * (want.abs() + float(want.square().mean().sqrt()))).all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_8_bit_cache_scores_of_zero_between_large_rows(cuda, kind):
    """q and k at right angles, whose scales' product alone is beyond F32."""
    c = Cache([5], 16, 8, 128, 3)
    k = torch.zeros((5, 8, 128), device=cuda)
    k[..., 1] = 2.0 ** 60
    v = torch.randn((5, 8, 128), device=cuda, generator=gen(6))
    c.fill(k, v, cumulative([5]))
    q = torch.zeros((1, 16, 128), device=cuda, dtype=DT[kind])
    q[..., 0] = 2.0 ** 120
    want = c.values(0)[1].mean(0).repeat_interleave(2, 0)
    got = B.flash_attn_paged_batch_q8(q, *c.args, c.table, c.seq_lens)[0].double()
    assert ((got - want).abs() <= UNIT[kind] * want.abs() + 1e-5 * (want.abs() + float(want.square().mean().sqrt()))).all()


def pool(x, block=16):
    n = -(-x.shape[0] // block)
    p = torch.zeros((n, block) + x.shape[1:], dtype=x.dtype, device=x.device)
    p.view(-1, *x.shape[1:])[:x.shape[0]] = x
    return p


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", [(16, 8, 128), (8, 4, 64)])
@pytest.mark.parametrize("n", [1, 300, 2500])
@pytest.mark.parametrize("seqs", [9, 150])
@pytest.mark.parametrize("target", TARGETS)
def test_shared_prefix(cuda, kind, layout, n, seqs, target):
    if not possible(kind, target):
        return
    q, k, v = rows(n, target, *layout, kind)
    kp, vp = pool(k), pool(v)
    table = torch.arange(kp.shape[0], dtype=torch.int32, device=cuda)[None]
    own = torch.zeros((seqs, 1), dtype=torch.int32, device=cuda)  # the first key again, of some
    lens = [s % 2 if n > 1 else 0 for s in range(seqs)]
    got = B.flash_attn_paged_shared(q.expand(seqs, -1, -1).contiguous(), kp, vp, table, ints([n]), ints([0, seqs]), own, ints(lens))
    close(got, v[min(3, n - 1)].repeat_interleave(layout[0] // layout[1], 0), kind)


@pytest.mark.parametrize("layout", [(16, 8, 128), (8, 4, 64)])
@pytest.mark.parametrize("n", [300, 2500])
@pytest.mark.parametrize("target", TARGETS)
def test_packed_f32(cuda, layout, n, target):
    """Queries of a prompt's end, each behind the deciding key."""
    q, k, v = rows(n, target, *layout, "f32")
    got = B.flash_attn_packed(q.expand(200, -1, -1).contiguous(), k, v, ints([0, 200]), ints([0, n]))
    close(got, v[3].repeat_interleave(2, 0), "f32")
