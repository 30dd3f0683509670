"""Workspaces of the 8-bit decode and of shared-prefix attention: calls without enough of one are refused, and one for many
sequences does for fewer (no GPU: a refused call touches no pointer)."""

import pytest

import b200infer.capi as L
from test_step_refusals import INVALID, P, decode, pool, shared


def test_decode_refuses_what_is_too_small():
    need = L.lib().b200_flash_attn_paged_batch_q8_workspace_bytes(200, 64, 64, 4, 2)
    assert need > 0
    assert decode(n=200, ws=None) == INVALID and decode(n=200, wsb=need - 1) == INVALID and decode(n=200, ws=P + 4) == INVALID


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("n,groups,blocks,pblocks", [
    (200, 2, 4, 4),       # many short sequences
    (2, 1, 4, 512),       # few behind a long prefix (F32: planes)
    (1, 1, 300, 4),       # one with a wide table of its own
    (300, 0, 4, 4)])      # no group
def test_shared_refuses_what_is_too_small(dtype, n, groups, blocks, pblocks):
    need = L.lib().b200_flash_attn_paged_shared_workspace_bytes(n, blocks * 16, groups, pblocks * 16 if groups else 0, 64, 4, 2, dtype)
    assert need > 0
    args = dict(n=n, groups=groups, stride=blocks, blocks=blocks, pstride=pblocks, pblocks=pblocks)
    p = pool(dtype=dtype)
    assert shared(p, **args, ws=None) == INVALID
    assert shared(p, **args, wsb=need - 1) == INVALID
    assert shared(p, **args, ws=P + 4) == INVALID
    assert shared(p, **args, wsb=0) == INVALID


@pytest.mark.parametrize("heads", [(32, 8), (16, 8), (16, 1), (150, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_f32_workspace_for_many_sequences_does_for_fewer(heads, D):
    """With planes too, at one number of groups."""
    size = L.lib().b200_flash_attn_paged_shared_workspace_bytes
    for keys, groups, prefix in ((1024, 1, 8192), (4096, 4, 1000), (16, 1, 100000), (64, 7, 2048), (64, 2, 2049), (4000, 1, 97)):
        sizes = [size(n, keys, groups, prefix, D, *heads, 0) for n in list(range(1, 300)) + [500, 5000]]
        assert sizes == sorted(sizes)
