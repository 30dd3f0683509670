"""Append and read back of rows at both ends of the exponents' range, as the header states them: elements that round to 2^128
read as infinite, and BF16 rounds multiples of less than 2^-133."""
import math

import pytest
import torch

import b200infer as B
from test_gpu_q8 import DT, Cache, cumulative, held

pytestmark = pytest.mark.gpu


def through(x, kind):
    """(what the read gives, the exact values held) of rows x (n, 1, 64)."""
    c = Cache([len(x)], 16, 1, x.shape[2], 7)
    cu = cumulative([len(x)])
    c.fill(x, x, cu)
    q, b = held(x)
    k, v = B.paged_kv_read_q8(cu, c.seq_lens, len(x), *c.args, c.table, dtype=DT[kind])
    assert torch.equal(k, v)
    return k, q * torch.exp2(b.double() - 127.0)[..., None]


@pytest.mark.parametrize("source", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_largest_rows(cuda, source, kind):
    most = torch.finfo(DT[source]).max
    below = 248 * 2.0 ** 120 - (2.0 ** 104 if source == "f32" else 2.0 ** 120)  # the next smaller number
    x = torch.zeros((4, 1, 64), device=cuda, dtype=torch.float64)
    x[0, 0, :3] = torch.tensor([most, -most, 1e38], dtype=torch.float64)
    x[1, 0, :2] = torch.tensor([248 * 2.0 ** 120, 2.0 ** 120], dtype=torch.float64)
    x[2, 0, :2] = torch.tensor([below, -below], dtype=torch.float64)
    x[3, 0, :2] = torch.tensor([240 * 2.0 ** 120, 3.5 * 2.0 ** 119], dtype=torch.float64)
    x = x.to(DT[source])
    got, want = through(x, kind)
    assert got[0, 0, 0] == math.inf and got[0, 0, 1] == -math.inf and got[1, 0, 0] == math.inf
    finite = want.abs() < 2.0 ** 128
    assert torch.isfinite(got[finite].double()).all() and int((~finite).sum()) == 3
    assert torch.equal(got.double()[finite], want[finite])
    assert ((got.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs())[finite].all()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_smallest_rows(cuda, kind):
    """Rows near 2^-127, whose least elements are multiples of 2^-136."""
    x = torch.zeros((2, 1, 64), device=cuda)
    x[0, 0] = torch.arange(64, device=cuda) * 2.0 ** -136
    x[1, 0] = torch.arange(64, device=cuda) * 2.0 ** -130
    got, want = through(x, kind)
    assert torch.equal(got, want.to(DT[kind]))  # exact in F32, one rounding in BF16
    if kind == "bf16":
        assert got[0, 0, 1] == 0 and got[0, 0, 2] == 0 and got[0, 0, 8] == 2.0 ** -133
