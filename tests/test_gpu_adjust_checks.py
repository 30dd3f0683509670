"""b200_adjust_logits reports what makes no sense in a row's request whether or not the row's lists hold anything."""
import math

import pytest
import torch

import b200infer as B
from test_gpu_adjust_logits import BAD_LOGITS, BAD_POSITION, floats, gen, ints

pytestmark = pytest.mark.gpu

EMPTY = dict(dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("vocab", [100, 20000])
@pytest.mark.parametrize("kw", [dict(repetition=[1.0, 0.0]), dict(repetition=[1.0, -2.0]), dict(repetition=[1.0, math.nan]),
                                dict(repetition=[1.0, math.inf]), dict(frequency=[0.0, math.inf]), dict(presence=[0.0, math.nan])])
def test_bad_penalties_of_rows_without_history(cuda, vocab, kw):
    x = torch.randn((2, vocab), device=cuda, generator=gen(3))
    kw = {name: floats(v) for name, v in kw.items()}
    one = dict(bias_ids=ints([7]), bias_values=floats([2.0]))
    want = x.clone()
    want[1, 7] += 2.0
    for tokens, cu, more, out in (
            (ints([5]), [0, 1, 1], {}, x), (torch.empty(0, **EMPTY), [0, 0, 0], {}, x),
            (ints([5, vocab]), [0, 1, 2], {}, x),  # a history that names no token
            (torch.empty(0, **EMPTY), [0, 0, 0], dict(one, cu_bias=ints([0, 0, 1])), want)):
        status = ints([0])
        got = B.adjust_logits(x, tokens, ints(cu), status=status, **kw, **more)
        assert int(status) != 0 and (int(status) == BAD_LOGITS or vocab in tokens.tolist())
        assert torch.equal(got, out)


def test_good_penalties_of_rows_without_history(cuda):
    x = torch.randn((2, 5000), device=cuda, generator=gen(4))
    status = ints([0])
    got = B.adjust_logits(x, torch.empty(0, **EMPTY), ints([0, 0, 0]), ints([0, 0]), floats([1.2, 0.5]), floats([0.1, -0.1]),
                          floats([0.5, 0.0]), torch.empty(0, **EMPTY), floats([]), ints([0, 0, 0]), status=status)
    assert int(status) == 0 and torch.equal(got, x)


@pytest.mark.parametrize("cu", [[0, 5, 5], [0, 0, 1], [-1, 0, 0], [2, 1, 0]])
def test_offsets_of_empty_lists(cuda, cu):
    x = torch.randn((2, 300), device=cuda, generator=gen(5))
    none = torch.empty(0, **EMPTY)
    for kw in (dict(tokens=none, cu_tokens=ints(cu)), dict(bias_ids=none, bias_values=floats([]), cu_bias=ints(cu))):
        status = ints([0])
        assert torch.equal(B.adjust_logits(x, status=status, **kw), x)
        assert int(status) == BAD_POSITION
