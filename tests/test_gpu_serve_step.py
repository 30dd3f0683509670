"""The operators of a serving step together: the example with an 8-bit cache, behind a shared prefix and with adjusted
logits; whole steps in CUDA graphs; workspaces and streams that calls share.

Two ways to the same F32 logits differ by sums in different orders: within 1e-4 (rel_err), the bar of the engine's logits.
"""
import math

import pytest
import torch

import b200infer as B
from conftest import rel_err
from test_gpu_serve_batch import serve  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def prompts_of(d, lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, d.cfg.vocab, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("block_tokens,head", [(16, 100), (7, 33), (16, 1)])
def test_behind_a_prefix(cuda, serve, block_tokens, head):  # noqa: F811
    """Prompts behind a prefix that is cached once give the logits of the whole prompts."""
    d = serve.Decoder(serve.Config(layers=2), n_blocks=300, block_tokens=block_tokens)
    first, *tails = prompts_of(d, (head, 1, 40, 130))
    free = len(d.pages.free)
    prefix = d.prefix(first)
    got, lens = d.prefill(tails, prefix)
    steps = [got]
    for i in range(4):
        lens = [n + 1 for n in lens]
        steps.append(d.step(torch.tensor([7 * i, 11, 5 + i], dtype=torch.int32).cuda(), lens, prefix))
    for s in range(3):
        d.pages.release(s)
    prefix.release()
    assert len(d.pages.free) == free and int(d.status) == 0
    want, lens = d.prefill([first + t for t in tails])
    assert rel_err(steps[0].cpu().numpy(), want.cpu().numpy()) <= 1e-4
    for i in range(4):
        lens = [n + 1 for n in lens]
        want = d.step(torch.tensor([7 * i, 11, 5 + i], dtype=torch.int32).cuda(), lens)
        assert rel_err(steps[i + 1].cpu().numpy(), want.cpu().numpy()) <= 1e-4


def test_eight_bit_cache(cuda, serve):  # noqa: F811
    """Steps over the 8-bit cache give the logits of attention, by its formula in float64, over what the cache reads as; so do
    prompts that go on behind a cached head."""
    d = serve.Decoder(serve.Config(layers=2), cache="q8")
    logits, lens = d.prefill(prompts_of(d, (3, 90, 17)))
    chunk = [[1, 2, 3], [5], [9, 8]]
    before = [t.view(torch.uint8).clone() for t in (d.pages.k, d.pages.v, d.pages.k_scale, d.pages.v_scale)]

    def by_formula(lens):
        table = d.pages.table[:3].cuda()

        def attend(q, k, v, cu, keys=None, status=None, **_):
            out = torch.empty_like(q)
            cu, keys = cu.tolist(), (cu if keys is None else keys).tolist()
            for s in range(3):
                kk, vv = (x[keys[s]:keys[s + 1]].double().repeat_interleave(2, 1) for x in (k, v))
                rows, n = q[cu[s]:cu[s + 1]].double(), keys[s + 1] - keys[s]
                a = torch.einsum("ihd,jhd->hij", rows, kk) / math.sqrt(d.cfg.dim)
                seen = torch.arange(n, device="cuda")[None] <= n - len(rows) + torch.arange(len(rows), device="cuda")[:, None]
                out[cu[s]:cu[s + 1]] = torch.einsum("hij,jhd->ihd", torch.softmax(a.masked_fill(~seen, -math.inf), -1), vv).float()
            return out

        def batch(q, kp, vp, ks, vs, tb, lens_dev, status=None):
            at = torch.tensor([0] + lens).cumsum(0).int().cuda()
            k, v = B.paged_kv_read_q8(at, lens_dev, sum(lens), kp, vp, ks, vs, table, dtype=torch.float32)
            return attend(q, k, v, torch.arange(4), at)

        return attend, batch

    real = B.flash_attn_packed, B.flash_attn_paged_batch_q8
    got = []
    for formula in (False, True):
        for t, b in zip((d.pages.k, d.pages.v, d.pages.k_scale, d.pages.v_scale), before):
            t.view(torch.uint8).copy_(b)
        try:
            longer = [n + len(c) for n, c in zip(lens, chunk)]
            if formula:
                B.flash_attn_packed, B.flash_attn_paged_batch_q8 = by_formula([n + 1 for n in longer])
            first, now = d.extend(chunk, lens)
            assert now == longer
            got.append((first, d.step(torch.tensor([4, 5, 6], dtype=torch.int32).cuda(), [n + 1 for n in now])))
        finally:
            B.flash_attn_packed, B.flash_attn_paged_batch_q8 = real
    assert int(d.status) == 0
    for a, b in zip(*got):
        # (the two caches' layers may hold an element one step apart where its value lies at a border)
        assert rel_err(a.cpu().numpy(), b.cpu().numpy()) <= 2e-2
        assert float((a - b).norm() / b.norm()) <= 1e-3


def test_generate_with_requests(cuda, serve):  # noqa: F811
    d = serve.Decoder(serve.Config(layers=2))
    prompts = [[5, 6, 7], list(range(100)), [9]]
    free = len(d.pages.free)
    plain = d.generate(prompts, 6)
    assert torch.equal(d.generate(prompts, 6, repetition=1.0, bias={}, allowed=torch.ones(d.cfg.vocab, dtype=torch.bool)), plain)
    # a token that may not be drawn, by bias or by mask, is not; others stay as they are until then
    for ban in (dict(bias={int(plain[0, 0]): -math.inf}),
                dict(allowed=torch.arange(d.cfg.vocab) != int(plain[0, 0]))):
        got = d.generate(prompts, 6, **ban)
        assert int(plain[0, 0]) not in got.flatten().tolist()
    only = torch.zeros(d.cfg.vocab, dtype=torch.bool)
    only[[17, 40]] = True
    assert set(d.generate(prompts, 6, allowed=only, temperature=1.0, seed=2).flatten().tolist()) <= {17, 40}
    # a presence penalty larger than any logit: no token twice
    got = d.generate(prompts, 6, presence=1e6)
    assert all(len(set(row)) == 6 for row in got.tolist())
    prefix = d.prefix([3, 1, 4, 1, 5])
    assert torch.equal(d.generate(prompts, 6, prefix=prefix), d.generate([prefix.tokens + p for p in prompts], 6))
    prefix.release()
    q8 = serve.Decoder(serve.Config(layers=2), cache="q8")
    assert torch.equal(q8.generate(prompts, 6, repetition=1.2), q8.generate(prompts, 6, repetition=1.2))
    assert len(d.pages.free) == free
    with pytest.raises(ValueError):
        q8.generate(prompts, 2, prefix=q8.prefix([1, 2]))


class Step:
    """A step's inputs at fixed addresses, and the calls of one layer and one draw."""

    def __init__(self, kind, n=6, Hq=8, Hkv=4, D=64, bt=16, blocks=20, vocab=5003, seed=5):
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.n, self.dt, self.vocab = n, kind, vocab

        def normal(*shape):
            return torch.randn(shape, device="cuda", generator=g).to(kind)

        self.q, self.k, self.v, self.logits = normal(n, Hq, D), normal(n, Hkv, D), normal(n, Hkv, D), normal(n, vocab)
        total = (n + 2) * blocks
        self.pools = [normal(total, bt, Hkv, D) for _ in range(2)]
        self.pools8 = [torch.zeros((total, bt, Hkv, D), dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2)]
        self.scales = [torch.zeros((total, Hkv, bt), dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu) for _ in range(2)]
        tables = torch.randperm(total, device="cuda", generator=g).int().view(n + 2, blocks)
        self.table, self.prefix_table = tables[:n], tables[n:]
        self.prefix_lens = torch.tensor([100, 33], dtype=torch.int32, device="cuda")
        self.groups = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
        self.cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        self.lens = torch.tensor([1, 17, 33, 64, 300, 5][:n], dtype=torch.int32, device="cuda")
        self.history = torch.randint(0, vocab, (n * 40,), device="cuda", generator=g).int()
        self.cu_history = torch.arange(n + 1, dtype=torch.int32, device="cuda") * 40
        self.ones = torch.full((n,), 1.2, device="cuda")
        self.u = torch.rand(n, device="cuda", generator=g)
        self.mask = torch.randint(-2 ** 31, 2 ** 31, (n, (vocab + 31) // 32), device="cuda", generator=g, dtype=torch.int64).int()

    def again(self, lens):
        for t in (self.q, self.k, self.v, self.logits):
            t.copy_(torch.randn(t.shape, device="cuda", generator=self.g))
        self.lens.copy_(torch.tensor(lens[:self.n]))
        self.prefix_lens.copy_(torch.tensor(lens[:2][::-1]))
        self.u.uniform_(generator=self.g)

    def run(self, workspace=None):
        B.paged_kv_append_q8(self.k, self.v, self.cu, self.lens, *self.pools8, *self.scales, self.table)
        kr, vr = B.paged_kv_read_q8(self.cu, self.lens, self.n, *self.pools8, *self.scales, self.table, dtype=self.dt)
        a = B.flash_attn_paged_batch_q8(self.q, *self.pools8, *self.scales, self.table, self.lens, workspace=workspace)
        b = B.flash_attn_paged_shared(self.q, *self.pools, self.prefix_table, self.prefix_lens, self.groups, self.table, self.lens,
                                      workspace=workspace)
        x = B.adjust_logits(self.logits, self.history, self.cu_history, None, self.ones, self.ones, self.ones, mask=self.mask)
        return kr, vr, a, b, x, B.sample(x, self.u, self.ones)

    def workspace(self):
        return torch.full((1 << 25,), 0xFF, dtype=torch.uint8, device="cuda")


LENGTHS = ([1, 17, 33, 64, 300, 5], [320, 320, 1, 1, 2, 100], [0, 0, 0, 0, 0, 0], [15, 16, 17, 31, 32, 319])


@pytest.mark.parametrize("kind", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,layout", [(6, (8, 4, 64)), (6, (16, 8, 128)), (1, (16, 1, 128))])
def test_steps_in_graphs(cuda, kind, n, layout):
    """Two captured steps that share one workspace, replayed in turn with other inputs and lengths, give what the calls give
    outside the graphs."""
    steps = [Step(kind, n, *layout, seed=s) for s in (5, 6)]
    ws = steps[0].workspace()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s in steps:
            s.run(ws)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for s in steps:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(s.run(ws))
    for lens in LENGTHS:
        for s in steps:
            s.again(lens)
        for _ in range(2):
            for g in graphs:
                g.replay()
        got = [[t.clone() for t in o] for o in outs]
        for s, o in zip(steps, got):
            for x, y in zip(o, s.run()):
                assert torch.equal(x.nan_to_num(), y.nan_to_num()) and torch.equal(x.isnan(), y.isnan())


def test_two_streams_at_once(cuda):
    """Steps on two streams at the same time, each with its own outputs and workspace."""
    steps = [Step(torch.bfloat16, 6, 16, 8, 128, seed=s) for s in (7, 8)]
    want = [s.run() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [[], []]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(steps, streams)):
            with torch.cuda.stream(st):
                got[i].append(s.run())
    torch.cuda.synchronize()
    for w, runs in zip(want, got):
        for r in runs:
            for x, y in zip(w, r):
                assert torch.equal(x, y)


def test_inputs_are_left_alone(cuda):
    s = Step(torch.float16)
    keep = [t.clone() for t in (s.q, s.k, s.v, s.logits, s.table, s.lens, s.history, s.mask, *s.pools)]
    s.run()
    for a, b in zip(keep, (s.q, s.k, s.v, s.logits, s.table, s.lens, s.history, s.mask, *s.pools)):
        assert torch.equal(a, b)
