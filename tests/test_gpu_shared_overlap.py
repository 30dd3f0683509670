"""Shared-prefix attention with offsets out of order, so that several groups name a sequence: its row is zero. A sequence that
one group names sees that group's prefix (or is zero, where overlapping groups have more tiles than any ascending offsets), one
that none names its own positions; nothing hangs on the kernels' timing, the workspace's old content or the kernel that runs.
Bounds as in test_gpu_shared.py."""
import pytest
import torch

import b200infer as B
from test_gpu_shared import BAD_POSITION, DT, Batch, check, ints

pytestmark = pytest.mark.gpu


def batch(prefix, cu, layout, kind, n, block=16):
    b = Batch(prefix, [n] + [0] * (len(prefix) - 1), [(i * 7) % 40 + 1 for i in range(n)], block, layout, kind, 29)
    b.cu = ints(cu)
    names = {s: [g for g in range(len(prefix)) if cu[g] >= 0 and cu[g] <= s < cu[g + 1] <= n] for s in range(n)}
    b.group = {s: g[0] for s, g in names.items() if len(g) == 1}
    b.several = torch.tensor([len(names[s]) > 1 for s in range(n)], device="cuda")
    b.none = torch.tensor([not names[s] for s in range(n)], device="cuda")
    return b


def run(b, kind, room=True):
    want, w = b.want()
    seen = []
    for fill in (0x3F, 0x00, 0xFF, 0x3F):  # 0x3F: numbers of 0.75 that would look like a part
        status = ints([0])
        ws = torch.full((1 << 27,), fill, dtype=torch.uint8, device="cuda")
        seen.append(B.flash_attn_paged_shared(*b.args(), workspace=ws, status=status))
        assert int(status) == BAD_POSITION
    for x in seen[1:]:
        assert torch.equal(x, seen[0])
    got = seen[0]
    assert (got[b.several] == 0).all()
    rows = ~b.several
    if not room:
        rows = rows & (b.none | ~(got == 0).flatten(1).all(1))
    check(got[rows], want[rows], w[rows], kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout,n", [("g16", 48), ("g4", 200), ("g20", 30), ("g2", 60), ("g2d64", 130)])
def test_groups_alike(cuda, kind, layout, n):
    end = n - 1
    b = batch([500, 60, 300, 60, 700], [0, end, 0, end, 0, end], layout, kind, n)
    assert b.several[:end].all() and b.none[end]
    run(b, kind)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("layout", ["g2", "g4", "g2d64", "g16"])
@pytest.mark.parametrize("prefix,cu,n", [([700, 20, 130], [0, 40, 25, 51], 51), ([130, 20, 700], [0, 45, 7, 51], 51),
                                         ([300, 50, 200], [0, 6, 4, 9], 9), ([300, 50, 200], [0, 3, 2, 4], 4),
                                         ([300, 50, 200], [3, 0, 2, 4], 4), ([2500, 20, 2600], [0, 90, 50, 130], 130)])
def test_some_sequences_of_several_groups(cuda, kind, layout, prefix, cu, n):
    # g16: groups of 45 and 44 sequences, and of 90 and 80, have more tiles of 8 or 16 sequences than there is room for
    run(batch(prefix, cu, layout, kind, n), kind, room=layout != "g16" or n <= 9)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("n", [4, 51])
def test_order_alone(cuda, kind, n):
    """Groups out of order that do not overlap: each sequence sees its group's prefix."""
    cu = [2, 3, 0, 2] if n == 4 else [40, 51, 0, 40]  # groups 0 and 2; the one between is out of order
    b = batch([300, 20, 130], cu, "g4", kind, n)
    assert not b.several.any()
    run(b, kind)


@pytest.mark.parametrize("layout", ["g2", "g2d64"])
def test_spread_magnitudes(cuda, layout):
    """F32 tiles that the tensor-core kernel does over."""
    b = batch([700, 20, 130], [0, 40, 25, 51], layout, "f32", 51)
    b.k[b.prefix_table[0, 5]] *= 2.0 ** -30
    b.k[b.prefix_table[2, 1]] *= 2.0 ** -30
    run(b, "f32")


@pytest.mark.parametrize("kind", list(DT))
def test_many_heads_share_keys(cuda, kind):
    b = batch([150, 20, 90], [0, 30, 20, 50], "g20", kind, 50)
    b.q = torch.randn((50, 150, 64), device=cuda, generator=torch.Generator(device=cuda).manual_seed(3)).to(DT[kind])
    run(b, kind, room=False)  # 142 tiles of 64 rows, where ascending offsets have 120 at most


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("n", [4, 51])
def test_bad_block_of_one_of_them(cuda, kind, n):
    """The rows of the group whose prefix names a bad block are zero too, no other."""
    cu = [0, 3, 2, 4] if n == 4 else [0, 40, 25, 51]
    b = batch([700, 20, 130], cu, "g4", kind, n)
    want, w = b.want()
    b.prefix_table[0, 3] = b.k.shape[0]
    got = B.flash_attn_paged_shared(*b.args())
    zero = torch.tensor([b.group.get(s) == 0 for s in range(n)], device=cuda) | b.several
    assert (got[zero] == 0).all()
    check(got[~zero], want[~zero], w[~zero], kind)
