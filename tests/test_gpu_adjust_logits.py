"""b200_adjust_logits against the same steps in float64. Bounds: three F32 operations of unit roundoff 2^-24 on terms no
larger than |x| r + |f| count + |p| + |bias|, then the output's one rounding (2^-11 F16, 2^-8 BF16, half their epsilon;
2^-25 for F16 below its normals). Tokens without penalty or bias, and masked ones, are exact."""
import math

import pytest
import torch

import b200infer as B

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
BAD_TOKEN, BAD_POSITION, BAD_LOGITS = 1, 2, 3


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def floats(x):
    return torch.tensor(x, dtype=torch.float32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def words(allowed):
    n, vocab = allowed.shape
    pad = torch.zeros((n, -vocab % 32), dtype=torch.bool, device=allowed.device)
    w = (torch.cat([allowed, pad], 1).view(n, -1, 32).long() << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def expected(x, history, prompt, r, f, p, biases, allowed):
    """Rows in float64 and the size of their terms. history: lists of ids; biases: lists of (id, value)."""
    y = x.double().clone()
    size = y.abs()
    for s in range(x.shape[0]):
        ids = [t for t in history[s] if 0 <= t < x.shape[1]] if history else []
        for t in set(ids):
            y[s, t] = y[s, t] / r[s] if y[s, t] > 0 else y[s, t] * r[s]
            size[s, t] = max(float(size[s, t]), abs(float(y[s, t])))
        drawn = [t for t in history[s][max(prompt[s], 0):] if 0 <= t < x.shape[1]] if history else []
        for t in set(drawn):
            y[s, t] -= f[s] * drawn.count(t) + p[s]
            size[s, t] += abs(f[s]) * drawn.count(t) + abs(p[s])
        for t, b in dict(biases[s]).items() if biases else ():
            y[s, t] += b
            size[s, t] += abs(b)
    if allowed is not None:
        y[~allowed] = -math.inf
    return y, size


def check(got, y, size, x):
    kind = next(k for k in DT if DT[k] == got.dtype)
    fine = torch.isfinite(y)
    g = got.double()
    assert torch.equal(g[~fine], y[~fine])
    same = fine & (y == x.double())
    assert torch.equal(g[same], y[same])
    bound = UNIT[kind] * y.abs() + 4 * 2.0 ** -24 * size + (2.0 ** -25 if kind == "f16" else 0)
    assert ((g - y).abs() <= bound)[fine].all()


def pack(lists):
    flat = [t for l in lists for t in l]
    cu = [0]
    for l in lists:
        cu.append(cu[-1] + len(l))
    return ints(flat), ints(cu)


def request(n, vocab, seed, most=200):
    g = torch.Generator().manual_seed(seed)

    def ids(k):
        return (torch.rand(k, generator=g) ** 3 * vocab).long().clamp(max=vocab - 1).tolist()

    history = [ids(int(torch.randint(0, most, (1,), generator=g)) if s % 3 else 0) for s in range(n)]
    prompt = [len(h) // (1 + s % 3) for s, h in enumerate(history)]
    r = [[1.0, 1.3, 0.7][s % 3] for s in range(n)]
    f = [[0.0, 0.25, -0.5][(s // 2) % 3] for s in range(n)]
    p = [[0.0, 0.6][s % 2] for s in range(n)]
    biases = [[(t, float(b)) for t, b in zip(ids(s % 7), torch.randn(s % 7, generator=g) * 3)] for s in range(n)]
    return history, prompt, r, f, p, biases


def call(x, history, prompt, r, f, p, biases, allowed, **kw):
    t, cu = pack(history)
    bi, cb = pack([[t for t, _ in b] for b in biases])
    bv = floats([v for b in biases for _, v in b])
    return B.adjust_logits(x, t, cu, ints(prompt), floats(r), floats(f), floats(p), bi, bv, cb,
                           None if allowed is None else words(allowed), **kw)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("n,vocab", [(1, 1), (1, 151936), (3, 37), (5, 1024), (4, 32003), (70, 8193), (2, 9000)])
@pytest.mark.parametrize("masked", [False, True])
def test_everything(cuda, kind, n, vocab, masked):
    x = (torch.randn((n, vocab), device=cuda, generator=gen(n)) * 4).to(DT[kind])
    req = request(n, vocab, vocab + n)
    allowed = None
    if masked:
        allowed = torch.rand((n, vocab), device=cuda, generator=gen(5)) < torch.tensor([0.0, 1.0, 0.5, 0.01], device=cuda)[torch.arange(n) % 4][:, None]
    y, size = expected(x, *req, allowed)
    keep = x.clone()
    check(call(x, *req, allowed), y, size, x)
    assert torch.equal(x, keep)
    check(call(x, *req, allowed, out=x), y, size, keep)  # in place


@pytest.mark.parametrize("which", ["repetition", "frequency", "presence", "bias", "mask", "nothing"])
def test_each_alone(cuda, which):
    n, vocab = 3, 5000
    x = torch.randn((n, vocab), device=cuda, generator=gen(8))
    history, prompt, r, f, p, biases = request(n, vocab, 3, 900)
    t, cu = pack(history)
    allowed = torch.rand((n, vocab), device=cuda, generator=gen(9)) < 0.5
    one, zero, none = [1.0] * n, [0.0] * n, [[]] * n
    if which == "repetition":  # without a prompt's length the whole history is drawn
        got, want = B.adjust_logits(x, t, cu, repetition=floats(r)), (history, [0] * n, r, zero, zero, none, None)
    elif which == "frequency":
        got, want = B.adjust_logits(x, t, cu, ints(prompt), frequency=floats(f)), (history, prompt, one, f, zero, none, None)
    elif which == "presence":
        got, want = B.adjust_logits(x, t, cu, presence=floats(p)), (history, [0] * n, one, zero, p, none, None)
    elif which == "bias":
        bi, cb = pack([[t for t, _ in b] for b in biases])
        got = B.adjust_logits(x, bias_ids=bi, bias_values=floats([v for b in biases for _, v in b]), cu_bias=cb)
        want = ([[]] * n, [0] * n, one, zero, zero, biases, None)
    elif which == "mask":
        got, want = B.adjust_logits(x, mask=words(allowed)), ([[]] * n, [0] * n, one, zero, zero, none, allowed)
    else:
        got, want = B.adjust_logits(x), ([[]] * n, [0] * n, one, zero, zero, none, None)
    check(got, *expected(x, *want), x)


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("offset,out_offset", [(0, 0), (1, 1), (3, 0), (2, 5)])
def test_rows_of_any_alignment(cuda, kind, offset, out_offset):
    n, vocab = 3, 4099
    wide = torch.randn((n, vocab + 11), device=cuda, generator=gen(10)).to(DT[kind])
    target = torch.full((n, vocab + 9), 77.0, device=cuda).to(DT[kind])
    x, out = wide[:, offset:offset + vocab], target[:, out_offset:out_offset + vocab]
    req = request(n, vocab, 12)
    allowed = torch.rand((n, vocab), device=cuda, generator=gen(11)) < 0.5
    check(call(x, *req, allowed, out=out), *expected(x, *req, allowed), x)
    assert (target[:, :out_offset] == 77).all() and (target[:, out_offset + vocab:] == 77).all()


def test_one_row_and_one_mask_for_all(cuda):
    n, vocab = 4, 3001
    x = torch.randn((1, vocab), device=cuda, generator=gen(13)).expand(n, vocab)
    req = request(n, vocab, 14)
    allowed = (torch.rand((1, vocab), device=cuda, generator=gen(15)) < 0.3)
    t, cu = pack(req[0])
    got = B.adjust_logits(x, t, cu, ints(req[1]), floats(req[2]), floats(req[3]), floats(req[4]), mask=words(allowed).expand(n, -1))
    check(got, *expected(x, *req[:5], [[]] * n, allowed.expand(n, vocab)), x)


@pytest.mark.parametrize("kind", list(DT))
def test_values(cuda, kind):
    """Infinities and NaN: penalties act on them as arithmetic does, a mask hides them, a bias may forbid or force."""
    x = torch.zeros((1, 64), device=cuda, dtype=DT[kind])
    x[0, :6] = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 1.0, -1.0], dtype=DT[kind])
    x[0, 10], x[0, 11] = math.nan, math.inf
    allowed = torch.ones((1, 64), dtype=torch.bool, device=cuda)
    allowed[0, 10:13] = False
    got = B.adjust_logits(x, ints([0, 1, 2, 3, 4, 5, 4]), ints([0, 7]), None, floats([2.0]), floats([0.25]), floats([0.5]),
                          ints([20, 21, 22, 22]), floats([math.inf, -math.inf, 3.0, -2.0]), ints([0, 4]), words(allowed))[0].float()
    assert got[0] == math.inf and got[1] == -math.inf and torch.isnan(got[2])
    assert got[3] == -0.75 and got[4] == 0.5 - 1.0 and got[5] == -2.75
    assert (got[10:13] == -math.inf).all()
    assert got[20] == math.inf and got[21] == -math.inf and got[22] == -2.0  # the last of two
    assert (got[23:] == 0).all() and torch.isfinite(got[23:]).all()


def test_many_occurrences_are_counted(cuda):
    """A token drawn 100000 times, histories much longer than a chunk of the vocabulary."""
    vocab = 20000
    x = torch.randn((2, vocab), device=cuda, generator=gen(17))
    t = torch.randint(0, vocab, (150000,), device=cuda, generator=gen(18)).to(torch.int32)
    t[:100000] = 12345
    cu = ints([0, 149000, 150000])
    got = B.adjust_logits(x, t, cu, frequency=floats([0.125, 0.5]))
    for s in range(2):
        count = torch.bincount(t[int(cu[s]):int(cu[s + 1])].long(), minlength=vocab).double()
        want = x[s].double() - [0.125, 0.5][s] * count
        assert ((got[s].double() - want).abs() <= 2.0 ** -24 * (want.abs() + x[s].double().abs() + want.abs())).all()


def test_out_of_range(cuda):
    """Ids and offsets out of range are left out and reported; so is a penalty that makes no sense."""
    x = torch.randn((3, 100), device=cuda, generator=gen(19))
    status = ints([0])
    got = B.adjust_logits(x, ints([5, -1, 100, 2 ** 31 - 1, 7]), ints([0, 4, 4, 5]), presence=floats([1.0] * 3), status=status)
    assert int(status) == BAD_TOKEN
    check(got, *expected(x, [[5], [], [7]], [0] * 3, [1.0] * 3, [0.0] * 3, [1.0] * 3, None, None), x)
    status.zero_()
    got = B.adjust_logits(x, bias_ids=ints([5, -1, 100]), bias_values=floats([1.0, 2.0, 3.0]), cu_bias=ints([0, 3, 3, 3]), status=status)
    assert int(status) == BAD_TOKEN
    check(got, *expected(x, None, None, None, None, None, [[(5, 1.0)], [], []], None), x)
    for cu in ([0, 4, 2, 5], [-1, 1, 2, 5], [0, 1, 2, 6], [3, 1, 1, 5]):
        status.zero_()
        got = B.adjust_logits(x, ints([5, 6, 7, 8, 9]), ints(cu), presence=floats([1.0] * 3), status=status)
        assert int(status) == BAD_POSITION
        rows = [list(range(5 + a, 5 + b)) if 0 <= a <= b <= 5 else [] for a, b in zip(cu, cu[1:])]
        check(got, *expected(x, rows, [0] * 3, [1.0] * 3, [0.0] * 3, [1.0] * 3, None, None), x)
    for kw in (dict(repetition=floats([0.0, -1.0, math.inf])), dict(repetition=floats([math.nan] * 3)),
               dict(frequency=floats([math.inf] * 3)), dict(presence=floats([math.nan] * 3))):
        status.zero_()
        assert torch.equal(B.adjust_logits(x, ints([1, 2, 3]), ints([0, 1, 2, 3]), status=status, **kw), x)
        assert int(status) == BAD_LOGITS


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("vocab", [4089, 4093, 4094, 4095, 4096, 8191, 16379, 16383])
@pytest.mark.parametrize("n", [1, 600])
def test_ids_behind_a_row_that_ends_with_a_chunk(cuda, kind, vocab, n):
    """Ids past the vocabulary touch neither their row nor what lies behind it, where a chunk begins behind the row's end too."""
    x = torch.randn((n + 8, vocab), device=cuda, generator=gen(23)).to(DT[kind])
    out = torch.full_like(x, 7.0)
    ids = [vocab, vocab + 1, vocab + 100, vocab + 5000, 2 ** 31 - 1, -1, -2 ** 31, 3]
    t, cu = pack([ids] * n)
    status = ints([0])
    B.adjust_logits(x[:n], t, cu, presence=floats([1.0] * n), bias_ids=t, bias_values=floats([2.0] * len(t)), cu_bias=cu,
                    out=out[:n], status=status)
    assert int(status) == BAD_TOKEN
    check(out[:n], *expected(x[:n], [[3]] * n, [0] * n, [1.0] * n, [0.0] * n, [1.0] * n, [[(3, 2.0)]] * n, None), x[:n])
    assert (out[n:] == 7.0).all()


def test_prompt_lengths_past_the_history(cuda):
    x = torch.randn((3, 50), device=cuda, generator=gen(20))
    h = [[1, 1, 2], [3], [4, 4]]
    t, cu = pack(h)
    got = B.adjust_logits(x, t, cu, ints([2 ** 31 - 1, -5, 1]), floats([1.5] * 3), floats([0.5] * 3), floats([0.25] * 3))
    check(got, *expected(x, h, [2 ** 31 - 1, 0, 1], [1.5] * 3, [0.5] * 3, [0.25] * 3, None, None), x)


def test_a_row_without_allowed_tokens_cannot_be_sampled(cuda):
    x = torch.randn((2, 1000), device=cuda, generator=gen(21))
    allowed = torch.zeros((2, 1000), dtype=torch.bool, device=cuda)
    allowed[1, 123] = True
    y = B.adjust_logits(x, mask=words(allowed))
    status = ints([0])
    ids = B.sample(y, floats([0.3, 0.9]), floats([1.0, 0.0]), status=status)
    assert ids.tolist() == [-1, 123] and int(status) == BAD_LOGITS


def test_argument_errors(cuda):
    x = torch.zeros((2, 40), device=cuda)
    t, cu = ints([1]), ints([0, 1, 1])
    for kw in (dict(tokens=t), dict(cu_tokens=cu), dict(bias_ids=t), dict(tokens=t.long(), cu_tokens=cu), dict(tokens=t, cu_tokens=cu[:2]),
               dict(mask=ints([[0], [0]])), dict(mask=ints([[0, 0]])), dict(out=x.half()), dict(out=x[:1]),
               dict(tokens=t, cu_tokens=cu, repetition=floats([1.0]))):
        with pytest.raises((ValueError, TypeError)):
            B.adjust_logits(x, **kw)
    with pytest.raises(B.B200Error):
        B.adjust_logits(x, repetition=floats([1.0, 1.0]))
    assert B.adjust_logits(x[:0]).shape == (0, 40)
