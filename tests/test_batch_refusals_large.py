"""Host-side checks of the batched serving entry points at sizes whose products pass 64 bits or
whose indexes pass 31 (no GPU: a refused call touches no pointer)."""
import pytest

from test_batch_refusals import UNSUPPORTED, append, decode, packed, pool


@pytest.mark.parametrize("kw", [dict(tq=2 ** 62, Hq=8), dict(tq=2 ** 61, Hq=16), dict(n=2 ** 31 - 100), dict(tq=2 ** 30, Hq=4)])
def test_packed_sizes(kw):
    assert packed(**kw) == UNSUPPORTED


@pytest.mark.parametrize("kw", [dict(n_head_kv=2 ** 44, head_dim=2 ** 20), dict(n_head_kv=2 ** 60, head_dim=16),
                                dict(n_head_kv=2 ** 20, head_dim=128)])
def test_append_row_sizes(kw):
    assert append(pool(**kw)) == UNSUPPORTED


def test_sequence_counts():
    assert append(n=2 ** 31 - 100) == UNSUPPORTED and append(t=2 ** 31 - 100) == UNSUPPORTED
    assert decode(n=2 ** 31 - 100) == UNSUPPORTED
