"""8-bit append of rows whose offsets pass the rows that there are: reported and left out, as the read does."""
import pytest
import torch

import b200infer as B
from test_gpu_q8 import BAD_POSITION, DT, Cache, gen, held, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("heads", [(2, 64), (3, 128)])
@pytest.mark.parametrize("cu,good", [([0, 10, 40], 0), ([-3, 10, 30], 1), ([0, 12, 31], 0)])
def test_append_offsets_past_the_rows(cuda, kind, heads, cu, good):
    """Of two sequences of 50 positions one has offsets within the 30 rows; the other's are left as they were."""
    Hkv, D = heads
    c = Cache([50, 50], 8, Hkv, D, 3)
    rows = torch.randn((30, Hkv, D), device=cuda, generator=gen(4)).to(DT[kind])
    want = c.bytes()
    first, last = cu[good], cu[good + 1]
    page, place = c.places(good, 50 - (last - first), 50)
    y, b = held(rows[first:last])
    for q, e in ((0, 2), (1, 3)):
        want[q][page, place] = y.float().to(torch.float8_e4m3fn).view(torch.uint8)
        want[e][page, :, place] = b
    status = ints([0])
    B.paged_kv_append_q8(rows, rows, ints(cu), c.seq_lens, *c.args, c.table, status=status)
    for got, w in zip(c.bytes(), want):
        assert torch.equal(got, w)
    assert int(status) == BAD_POSITION
