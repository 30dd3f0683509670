"""The batch-serving example against the same decoder run one sequence at a time on the
contiguous single-sequence ops (b200_flash_attn), teacher-forced with the batch's tokens.

Both are F32 with sums in different orders: logits within 1e-4 (rel_err), the bar of the
engine's logits; greedy tokens equal wherever the two best logits are further apart than that.
"""
import importlib.util
import os

import pytest
import torch

import b200infer as B
from conftest import REPO, rel_err

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def serve():
    spec = importlib.util.spec_from_file_location("serve_batch", os.path.join(REPO, "examples", "serve_batch.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def single_logits(d, tokens):
    """Logits of every position of one sequence, contiguous ops only."""
    c = d.cfg
    ids = torch.tensor(tokens, dtype=torch.int32).cuda()
    pos = torch.arange(len(tokens), dtype=torch.int32).cuda()
    h = B.get_rows(d.embed, ids)
    T = len(tokens)
    for w in d.layers:
        x = B.rms_norm(h, d.norm, c.eps)
        q, k, v = (B.mul_mat(w[n], x).view(T, -1, c.dim) for n in "qkv")
        q, k, _ = B.qk_norm_rope(q, k, d.head_norm, d.head_norm, d.freq, pos, c.eps, c.ctx)
        h = B.add(h, B.mul_mat(w["o"], B.flash_attn(q, k, v, 0).view(T, -1)))
        x = B.rms_norm(h, d.norm, c.eps)
        h = B.add(h, B.mul_mat(w["down"], B.swiglu(B.mul_mat(w["gate"], x), B.mul_mat(w["up"], x))))
    return B.mul_mat(d.embed, B.rms_norm(h, d.norm, c.eps))


@pytest.mark.parametrize("block_tokens", [16, 7])
def test_batch_equals_single_sequences(cuda, serve, block_tokens):
    d = serve.Decoder(serve.Config(layers=2), n_blocks=300, block_tokens=block_tokens)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, d.cfg.vocab, (n,), generator=g).tolist() for n in (1, 200, 33, 130)]
    logits, lens = d.prefill(prompts)
    seqs = [list(p) for p in prompts]
    batch = [logits]
    for _ in range(6):
        tokens = logits.argmax(1).int()
        for s, t in zip(seqs, tokens.tolist()):
            s.append(t)
        lens = [n + 1 for n in lens]
        logits = d.step(tokens, lens)
        batch.append(logits)
    assert int(d.status) == 0
    for i, (p, s) in enumerate(zip(prompts, seqs)):
        want = single_logits(d, s)[len(p) - 1:]
        got = torch.stack([b[i] for b in batch])
        assert rel_err(got.cpu().numpy(), want.cpu().numpy()) <= 1e-4
        best = want.topk(2, 1)[0]
        clear = (best[:, 0] - best[:, 1]) > 1e-3 * want.abs().max()
        assert torch.equal(got.argmax(1)[clear], want.argmax(1)[clear])


def test_generate(cuda, serve):
    d = serve.Decoder(serve.Config(layers=2))
    prompts = [[5, 6, 7], list(range(100)), [9]]
    free = len(d.pages.free)
    greedy = d.generate(prompts, 5)
    assert torch.equal(greedy, d.generate(prompts, 5)) and len(d.pages.free) == free
    one = dict(temperature=0.9, top_k=40, top_p=0.9, min_p=0.02, seed=4)
    assert torch.equal(d.generate(prompts, 5, **one), d.generate(prompts, 5, **one))
    assert torch.equal(d.generate(prompts, 5, temperature=0.9, top_k=1), greedy)
