"""The weights of shared prefixes count with more bits than the cache's 16-bit type has, as those of a sequence's own keys do
(flash_attn_paged_batch): an answer does not lose bits where a prefix is shared, and depends on neither the tables' widths nor
the kernel that they choose.

Bound per output element with `want` exact, W1 = sum p_j |v_j| and W = sqrt(sum (p_j v_j)^2) over the keys: the output's one
rounding u |want|; a weight held as two numbers of the type is off by at most half of the second's last bit, 2^-18 (BF16) or
2^-24 (F16) of it, independently: at most 2^-18 W four times over; sums of tensor-core products that are cut, not rounded, to
24 bits, one a 16 keys and term: at most 2^-23 each, on half of the sum on average, keys / 16 2^-23 W1; 1e-5 of |want| + RMS
for exponentials, scores and joins; 2^-25 for F16 outputs below its normals. Weights rounded once to the type would move
an output by up to u W, which a scale that lets few keys decide makes far larger than that.
"""
import math

import pytest
import torch

import b200infer as B
from test_gpu_shared import DT, UNIT, Batch

pytestmark = pytest.mark.gpu

SCALE = 0.5  # scores of unit normal rows of 128: a standard deviation of 5.7


def exact(b, scale):
    out = []
    for s in range(len(b.own)):
        k, v = (x.double() for x in b.keys(s))
        rep = b.q.shape[1] // k.shape[1]
        k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
        p = torch.softmax(torch.einsum("hd,mhd->hm", b.q[s].double(), k) * scale, -1)
        out.append((torch.einsum("hm,mhd->hd", p, v), torch.einsum("hm,mhd->hd", p.square(), v.square()).sqrt(),
                    torch.einsum("hm,mhd->hd", p, v.abs()) * k.shape[0]))
    return (torch.stack(x) for x in zip(*out))


def check(got, b, kind, scale=SCALE):
    want, w, w1 = exact(b, scale)
    rms = float(want.square().mean().sqrt())
    bound = UNIT[kind] * want.abs() + 4 * 2.0 ** -18 * w + 2.0 ** -27 * w1 + 1e-5 * (want.abs() + rms) + (2.0 ** -25 if kind == "f16" else 0.0)
    worst = float(((got.double() - want).abs() / bound).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64", "g3", "g16"])
@pytest.mark.parametrize("prefix,seqs", [([700, 130], [40, 11]), ([2003], [70]), ([129] * 6, [7] * 6)])
def test_weights(cuda, kind, layout, prefix, seqs):
    n = sum(seqs)
    b = Batch(prefix, seqs, [(i * 29) % 60 for i in range(n)], 16, layout, kind, 31)
    check(B.flash_attn_paged_shared(*b.args(), scale=SCALE), b, kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_any_width_of_table(cuda, kind):
    """The same call by one launch and, with a table wider than it takes, by the prefixes' kernel."""
    b = Batch([301], [4], [3, 40, 17, 90], 16, "g2", kind, 33)
    check(B.flash_attn_paged_shared(*b.args(), scale=SCALE), b, kind)
    wide = torch.full((1, 600), -1, dtype=torch.int32, device=cuda)
    wide[:, :b.prefix_table.shape[1]] = b.prefix_table
    b.prefix_table = wide
    check(B.flash_attn_paged_shared(*b.args(), scale=SCALE), b, kind)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_as_exact_as_without_sharing(cuda, kind):
    """Against the batched decode over tables that name the prefix's blocks first: errors of the same size."""
    b = Batch([2048], [40], [(i * 37) % 300 for i in range(40)], 16, "g4", kind, 35)
    table = torch.cat([b.prefix_table.expand(40, -1), b.table], 1).contiguous()
    lens = torch.tensor([2048 + n for n in b.own], dtype=torch.int32, device=cuda)
    want = next(exact(b, 1 / math.sqrt(128)))
    off = [float((x.double() - want).norm() / want.norm()) for x in (
        B.flash_attn_paged_shared(*b.args()), B.flash_attn_paged_batch(b.q, b.k, b.v, table, lens))]
    assert off[0] <= 1.1 * off[1], off
    assert DT[kind] == b.q.dtype
