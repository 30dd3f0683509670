"""b200_sample against its definition in float64 / exact integers on the host.

The kernel's weights are floor(2^40 e) with e the F32 exponential of the F32 product
(x - max) * (1 / T), which here is evaluated in float64 from the same F32 product: e then
differs by the error of the F32 exponential, at most 2 units in its last place (2^-22
relative). Every threshold and every running sum therefore lies within 2^-22 relative, and the
tests draw u and the filters where the exact answer does not change within 2^-20 (a row that
comes closer than that to an edge may give any token up to the one past the edge).
"""
import math

import numpy as np
import pytest
import torch

import b200infer as B

pytestmark = pytest.mark.gpu
EDGE = 2.0 ** -20


def answers(x, temp, top_k, top_p, min_p, u):
    """Token ids that the definition allows when every sum may move by EDGE, relative."""
    x = np.asarray(x, np.float32)
    V = len(x)
    top = x.max()
    if temp <= 0:
        return {int(x.argmax())}
    inv = np.float32(1) / np.float32(temp)
    w = np.floor(np.exp(((x - top) * inv).astype(np.float64)) * 2.0 ** 40)
    order = np.lexsort((np.arange(V), -x.astype(np.float64)))
    ids = set()
    for slack_p in (-EDGE, EDGE):
        n = V if top_k <= 0 else min(top_k, V)
        head = order[:n]
        if top_p < 1:
            run = np.cumsum(w[head])
            n = 1 + int(np.searchsorted(run, math.floor(top_p * run[-1] * (1 + slack_p)), side="left"))
            head = head[:n]
        for slack_m in (-EDGE, EDGE):
            kept = head[w[head] >= min(min_p, 1.0) * 2.0 ** 40 * (1 + slack_m)] if min_p > 0 else head
            kept = np.sort(kept)
            if len(kept) == 0:
                continue
            run = np.cumsum(w[kept])
            first, last = (np.searchsorted(run, min(max(math.floor(u * run[-1]) + slack * run[-1], 0), run[-1] - 1),
                                           side="right") for slack in (-EDGE, EDGE))
            ids.update(int(i) for i in kept[first:last + 1])
    return ids


def draw(x, temp, top_k, top_p, min_p, u, **kw):
    n = x.shape[0]
    f = lambda v, kind: torch.as_tensor(np.broadcast_to(v, (n,)).copy(), dtype=kind).cuda()  # noqa: E731
    return B.sample(x, f(u, torch.float32), f(temp, torch.float32), None if top_k is None else f(top_k, torch.int32),
                    None if top_p is None else f(top_p, torch.float32), None if min_p is None else f(min_p, torch.float32),
                    **kw).cpu().numpy()


def logits(n, vocab, kind, seed, sigma=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((n, vocab), device="cuda", generator=g) * sigma
    x[:, :: max(1, vocab // 7)] += 5
    return x.to(kind)


def check(x, temp, top_k, top_p, min_p, u, got):
    n = x.shape[0]
    h = x.float().cpu().numpy()
    bc = lambda v, d: np.broadcast_to(d if v is None else v, (n,))  # noqa: E731
    t, k, p, m, uu = bc(temp, 1), bc(top_k, 0), bc(top_p, 1.0), bc(min_p, 0.0), bc(u, 0)
    for i in range(n):
        ok = answers(h[i], np.float32(t[i]), int(k[i]), float(np.float32(p[i])), float(np.float32(m[i])),
                     float(np.float32(uu[i])))
        assert int(got[i]) in ok, (i, int(got[i]), ok)


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 512, 1000, 5003, 32003, 151936])
def test_filters(cuda, kind, vocab):
    n = 24
    rng = np.random.default_rng(vocab)
    x = logits(n, vocab, kind, vocab)
    temp = rng.choice([0.0, 0.5, 0.8, 1.0, 1.7], n).astype(np.float32)
    top_k = rng.choice([0, 1, 5, 50, 700, 10 ** 6], n).astype(np.int32)
    top_p = rng.choice([0.0, 0.3, 0.9, 0.99, 1.0], n).astype(np.float32)
    min_p = rng.choice([0.0, 0.02, 0.3, 1.0], n).astype(np.float32)
    u = rng.random(n).astype(np.float32)
    check(x, temp, top_k, top_p, min_p, u, draw(x, temp, top_k, top_p, min_p, u))
    for args in ((temp, None, None, None), (temp, top_k, None, None), (temp, None, top_p, None), (temp, None, None, min_p)):
        check(x, *args, u, draw(x, *args, u))


@pytest.mark.parametrize("kind,vocab", [(torch.float32, 600001), (torch.bfloat16, 1000003), (torch.float16, 2 ** 21)])
def test_vocabularies_past_shared_memory(cuda, kind, vocab):
    """Rows too long to be held on chip, which start at any element."""
    n = 4
    x = logits(n, vocab + 1, kind, vocab)[:, 1:]
    u = np.array([0.02, 0.4, 0.77, 0.995], np.float32)
    for args in ((1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.8, 40, 0.9, 0.01), (1.3, 0, 0.9, 0.0), (0.9, 5000, 0.95, 0.02)):
        check(x, *args, u, draw(x, *args, u))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 3, 700, 20011, 151936, 600001])
def test_greedy_rows(cuda, kind, vocab):
    """Temperature 0: the first of the largest, wherever it is, among equal ones and zeros of both signs."""
    x = logits(6, vocab, kind, vocab)
    x[1, vocab - 1] = x[1].max()
    x[2] = -1.0
    x[2, vocab // 2], x[2, vocab - 1] = -0.0, 0.0
    x[3] = -math.inf
    x[3, vocab - 1] = -5.0
    x[4] = 7.0
    x[5, vocab // 3] = 50.0
    u = np.full(6, 0.5, np.float32)
    got = draw(x, 0.0, None, None, None, u)
    assert list(got) == [int(np.argmax(r)) for r in x.float().cpu().numpy()]


@pytest.mark.parametrize("rows", [1, 3, 20, 40, 80, 160, 700])
def test_row_counts(cuda, rows):
    """Every cluster size gives the same token."""
    x = logits(1, 20011, torch.float32, 3).expand(rows, -1)
    for args in ((0.9, 40, 0.9, 0.01), (1.0, 0, 0.7, 0.0), (1.2, 0, 1.0, 0.0), (1.0, 900, 1.0, 0.0)):
        got = draw(x, *args, 0.61)
        assert (got == got[0]).all()
        check(x[:1], *args, 0.61, got[:1])


@pytest.mark.parametrize("vocab", [700, 40000, 300001])
def test_ties_and_flat_rows(cuda, vocab):
    """All logits equal, and a few values with many equal tokens: ties go by index, and a bin
    holds more tokens than are ranked directly."""
    flat = torch.zeros((4, vocab), device="cuda")
    u = np.array([0.0, 0.25, 0.5, 0.999], np.float32)
    k = 301
    got = draw(flat, 1.0, k, None, None, u)
    assert list(got) == [min(k - 1, int(np.float64(v) * k)) for v in u]
    check(flat, 1.0, 0, 0.5, 0.0, u, draw(flat, 1.0, None, 0.5, None, u))
    steps = (torch.arange(vocab, device="cuda") * 7919 % 5).float()[None].expand(4, -1).contiguous()
    for args in ((0.7, vocab // 3, 1.0, 0.0), (1.5, 0, 0.8, 0.0), (1.0, vocab // 2, 0.9, 0.1)):
        check(steps, *args, u, draw(steps, *args, u))
    close = 5 + torch.arange(vocab, device="cuda").float()[None].expand(4, -1) * 2.0 ** -20  # one narrow bin
    for args in ((1.0, vocab // 3, 1.0, 0.0), (1.0, 0, 0.37, 0.0)):
        check(close, *args, u, draw(close, *args, u))


@pytest.mark.parametrize("vocab", [700, 40000, 600001])
def test_short_top_k_in_odd_orders(cuda, vocab):
    """A short top-k whose tokens share their logits with many others, or lie side by side, descending or
    ascending along the row."""
    u = np.array([0.0, 0.3, 0.6, 0.999], np.float32)
    i = torch.arange(vocab, device="cuda").float()
    rows = (torch.zeros(vocab, device="cuda"), (i * 7919 % 5), -(i / 16).floor() * 0.03, (i / 400).floor() * 0.02,
            torch.where(i < 900, 9.0 + i * 2.0 ** -12, torch.sin(i)))
    for row in rows:
        x = row[None].expand(4, -1).contiguous()
        for args in ((0.9, 7, 1.0, 0.0), (1.0, 200, 0.8, 0.0), (1.3, 256, 1.0, 0.05), (0.7, 100, 0.95, 0.3)):
            check(x, *args, u, draw(x, *args, u))


@pytest.mark.parametrize("min_p", [1e-9, 1e-4, 0.02, 0.5, 1.0, 3.0])
def test_min_p_alone(cuda, min_p):
    x = logits(4, 50021, torch.float32, 31)
    x[1, :100] = x[1].max()
    u = np.array([0.001, 0.3, 0.6, 0.999], np.float32)
    for temp in (0.3, 1.0, 2.5):
        check(x, temp, 0, 1.0, min_p, u, draw(x, temp, None, None, min_p, u))


def test_masked_tokens_and_bad_rows(cuda):
    x = logits(8, 5000, torch.float32, 5)
    x[0, 100:] = -math.inf
    x[1] = -math.inf
    x[1, 4321] = -2.0
    x[2] = -math.inf                        # nothing to draw
    x[3, 17] = math.nan
    x[4, 4999] = math.inf
    x[5, :2500] = torch.finfo(torch.float32).min
    x[6] = torch.finfo(torch.float32).min   # the type's lowest value everywhere: a flat row
    u = np.full(8, 0.37, np.float32)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    for args in ((1.0, None, None, None), (0.8, 30, 0.9, 0.01)):
        status.zero_()
        got = draw(x, *args, u, status=status)
        assert int(status) == 3  # B200_DEV_BAD_LOGITS
        assert list(got[2:5]) == [-1, -1, -1] and got[1] == 4321 and 0 <= got[0] < 100 and got[5] >= 2500
        for i in (0, 1, 5, 6, 7):
            check(x[i:i + 1], *args, u[i:i + 1], got[i:i + 1])
    greedy = draw(x, 0.0, None, None, None, u)
    assert greedy[0] == int(x[0].argmax()) and greedy[1] == 4321 and greedy[6] == 0 and list(greedy[2:5]) == [-1, -1, -1]


def test_parameters_at_their_ends(cuda):
    x = logits(1, 3000, torch.float32, 6).expand(9, -1)
    best = int(x[0].argmax())
    last = int(torch.where(x[0] > x[0].max() - 20)[0][-1])
    f32 = np.float32
    temp = np.array([-1.0, 1e-42, 1e-30, np.inf, 1, 1, 1, np.nan, 1], f32)
    u = np.array([0.5, 0.5, 0.5, 0.0, 1.0, -3.0, 7.0, 0.5, np.nan], f32)
    got = draw(x, temp, None, None, None, u)
    assert list(got[:4]) == [best, best, best, 0]
    assert got[4] >= last and got[5] == 0 and got[6] == got[4] and list(got[7:]) == [-1, -1]
    u = np.full(9, 0.5, f32)
    assert (draw(x, 1.0, 1, None, None, u) == best).all() and (draw(x, 1.0, None, 0.0, None, u) == best).all()
    assert (draw(x, 1.0, None, None, 5.0, u) == best).all() and (draw(x, 1.0, -7, 2.0, -1.0, u) == draw(x, 1.0, None, None, None, u)).all()
    assert (draw(x, 1.0, None, math.nan, None, u) == -1).all()


def test_draws_follow_the_weights(cuda):
    """A grid of u over one row gives each token its share."""
    n = 4096
    x = logits(1, 300, torch.float32, 8).expand(n, -1)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = draw(x, 1.0, None, None, None, u)
    assert (np.diff(got) >= 0).all()  # by index
    p = torch.softmax(x[0].double(), 0).cpu().numpy()
    assert np.abs(np.bincount(got, minlength=300) / n - p).max() <= 1.01 / n + 2.0 ** -20


def test_strides_and_alignment(cuda):
    wide = logits(5, 4100, torch.bfloat16, 9)
    for off, width in ((0, 4100), (1, 4093), (3, 1001)):
        x = wide[:, off:off + width]
        u = np.linspace(0.05, 0.95, 5).astype(np.float32)
        check(x, 1.0, 20, 0.9, 0.0, u, draw(x, 1.0, 20, 0.9, 0.0, u))


def test_plain_form_agrees_bit_for_bit(cuda):
    """The weights use the F32 exponential that torch uses, so the plain integer form of the
    same definition gives the same tokens."""
    n, vocab = 64, 50021
    x = logits(n, vocab, torch.float32, 10)
    u = torch.rand(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    t = torch.full((n,), 0.9, device="cuda")
    w = torch.floor(torch.exp((x - x.amax(1, keepdim=True)) * (1.0 / t)[:, None]) * 2.0 ** 40).long()
    run = w.cumsum(1)
    at = (u.double()[:, None] * run[:, -1:].double()).long()
    assert torch.equal(B.sample(x, u, t), (run <= at).sum(1).int())


def test_refusals(cuda):
    x = torch.zeros((4, 100), device="cuda")
    one = torch.ones(4, device="cuda")
    for call in (lambda: B.sample(x.double(), one, one), lambda: B.sample(x, one[:3], one), lambda: B.sample(x, one, one.half()),
                 lambda: B.sample(x, one, one, top_k=one), lambda: B.sample(x.t(), one, one), lambda: B.sample(x, one.cpu(), one),
                 lambda: B.sample(x[0], one, one)):
        with pytest.raises((ValueError, TypeError)):
            call()
    with pytest.raises(B.B200Error) as e:
        B.sample(torch.zeros((1, 2 ** 21 + 1), device="cuda"), one[:1], one[:1])
    assert e.value.status == 2
    assert B.sample(x[:0], one[:0], one[:0]).numel() == 0
