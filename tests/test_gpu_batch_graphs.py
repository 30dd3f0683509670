"""The batched serving calls in CUDA graphs, and the packed attention's widest head groups."""
import pytest
import torch

import b200infer as B
from test_gpu_batch import DT, check, cumulative, gen, packed_exact

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", list(DT))
@pytest.mark.parametrize("group", [64, 65, 100, 128, 129, 200])
@pytest.mark.parametrize("lens", [([40, 1, 0, 7], [40, 300, 3, 2]), ([3], [2500])], ids=["ragged", "few_rows"])
def test_many_heads_share_keys(cuda, kind, group, lens):
    ql, kl = lens
    g = gen(51)
    q = torch.randn((sum(ql), 2 * group, 64), device=cuda, generator=g).to(DT[kind])
    k, v = (torch.randn((sum(kl), 2, 64), device=cuda, generator=g).to(DT[kind]) for _ in range(2))
    want, w = packed_exact(q, k, v, ql, kl)
    check(B.flash_attn_packed(q, k, v, cumulative(ql), cumulative(kl)), want, w, kind, True)


@pytest.mark.parametrize("kind", list(DT))
def test_a_step_in_a_graph(cuda, kind):
    """Append, both attentions and sampling, captured once; replays with other inputs and lengths
    give what the calls give outside the graph."""
    n, Hq, Hkv, D, bt, blocks, vocab = 5, 8, 4, 64, 16, 40, 5003
    g = gen(52)
    dt = DT[kind]

    def normal(*shape):
        return torch.randn(shape, device=cuda, generator=g).to(dt)

    T = 400
    s = dict(q=normal(T, Hq, D), k=normal(T, Hkv, D), v=normal(T, Hkv, D), q1=normal(n, Hq, D), logits=normal(n, vocab),
             u=torch.rand(n, device=cuda, generator=g), cu=cumulative([100, 50, 0, 200, 50]),
             lens=torch.tensor([100, 50, 0, 200, 50], dtype=torch.int32, device=cuda))
    pools = [torch.zeros((n * blocks, bt, Hkv, D), device=cuda, dtype=dt) for _ in range(2)]
    table = torch.randperm(n * blocks, device=cuda, generator=g).int().view(n, blocks)
    t, p = torch.full((n,), 0.8, device=cuda), torch.full((n,), 0.9, device=cuda)
    kk = torch.full((n,), 40, dtype=torch.int32, device=cuda)

    def step():
        B.paged_kv_append(s["k"], s["v"], s["cu"], s["lens"], *pools, table)
        return (B.flash_attn_packed(s["q"], s["k"], s["v"], s["cu"]),
                B.flash_attn_paged_batch(s["q1"], *pools, table, s["lens"]), B.sample(s["logits"], s["u"], t, kk, p))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for lens in ([100, 50, 0, 200, 50], [1, 0, 399, 0, 0], [80, 80, 80, 80, 80]):
        for name in ("q", "k", "v", "q1", "logits"):
            s[name].copy_(torch.randn(s[name].shape, device=cuda, generator=g))
        s["u"].uniform_(generator=g)
        s["lens"].copy_(torch.tensor(lens))
        s["cu"].copy_(cumulative(lens))
        for _ in range(2):
            graph.replay()
        copies = [x.clone() for x in got]
        for pool in pools:
            pool.zero_()
        for a, b in zip(copies, step()):
            assert torch.equal(a, b)
