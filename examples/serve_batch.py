"""Many sequences at once: prompts of different lengths are packed and prefilled together,
their K / V go into one paged cache, and every decode step attends, samples and appends for
all of them.

A Qwen3-shaped decoder with random weights on the single ops of the package (F32); with a
GPU: ``python examples/serve_batch.py``. ``Decoder.prefill`` and ``Decoder.step`` show how
flash_attn_packed, paged_kv_append, flash_attn_paged_batch and sample go together.
"""
import os
import sys
from dataclasses import dataclass

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "infer-llm_b200"))
import b200infer as B  # noqa: E402


@dataclass
class Config:
    vocab: int = 4096
    embd: int = 512
    layers: int = 4
    heads: int = 8
    heads_kv: int = 4
    dim: int = 64
    ff: int = 1024
    ctx: int = 2048
    theta: float = 1e6
    eps: float = 1e-6


class PagePool:
    """The free blocks of one paged cache (all layers use the same block numbers) and each
    sequence's table of them."""

    def __init__(self, cfg, n_blocks, block_tokens, max_seqs):
        self.bt = block_tokens
        self.free = list(range(n_blocks))[::-1]
        shape = (cfg.layers, n_blocks, block_tokens, cfg.heads_kv, cfg.dim)
        self.k = torch.empty(shape, device="cuda")
        self.v = torch.empty(shape, device="cuda")
        per_seq = -(-cfg.ctx // block_tokens)
        self.table = torch.full((max_seqs, per_seq), -1, dtype=torch.int32)
        self.owned = [[] for _ in range(max_seqs)]

    def grow(self, seq, tokens):
        """Blocks for `tokens` tokens of a sequence."""
        while len(self.owned[seq]) * self.bt < tokens:
            if not self.free:
                raise RuntimeError("the cache is full")
            block = self.free.pop()
            self.table[seq, len(self.owned[seq])] = block
            self.owned[seq].append(block)

    def release(self, seq):
        self.free += self.owned[seq]
        self.owned[seq] = []
        self.table[seq] = -1


class Decoder:
    def __init__(self, cfg, seed=0, n_blocks=512, block_tokens=16, max_seqs=16):
        self.cfg = cfg
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(n, k):
            return torch.randn((n, k), device="cuda", generator=g) * (1.0 / k ** 0.5)

        self.embed = weight(cfg.vocab, cfg.embd)
        self.norm = torch.ones(cfg.embd, device="cuda")
        self.head_norm = torch.ones(cfg.dim, device="cuda")
        self.layers = [dict(q=weight(cfg.heads * cfg.dim, cfg.embd), k=weight(cfg.heads_kv * cfg.dim, cfg.embd),
                            v=weight(cfg.heads_kv * cfg.dim, cfg.embd), o=weight(cfg.embd, cfg.heads * cfg.dim),
                            gate=weight(cfg.ff, cfg.embd), up=weight(cfg.ff, cfg.embd), down=weight(cfg.embd, cfg.ff))
                       for _ in range(cfg.layers)]
        self.freq = torch.from_numpy(B.rope_freqs(cfg.theta, cfg.dim)).cuda()
        self.pages = PagePool(cfg, n_blocks, block_tokens, max_seqs)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def _forward(self, ids, pos, cu_new, lens, table, attend):
        """Hidden rows of packed new tokens; `attend(layer, q, k, v)` is their attention."""
        c, h = self.cfg, B.get_rows(self.embed, ids)
        T = ids.numel()
        for n, w in enumerate(self.layers):
            x = B.rms_norm(h, self.norm, c.eps)
            q = B.mul_mat(w["q"], x).view(T, c.heads, c.dim)
            k = B.mul_mat(w["k"], x).view(T, c.heads_kv, c.dim)
            v = B.mul_mat(w["v"], x).view(T, c.heads_kv, c.dim)
            q, k, _ = B.qk_norm_rope(q, k, self.head_norm, self.head_norm, self.freq, pos, c.eps, c.ctx)
            B.paged_kv_append(k, v, cu_new, lens, self.pages.k[n], self.pages.v[n], table, status=self.status)
            h = B.add(h, B.mul_mat(w["o"], attend(n, q, k, v).view(T, -1)))
            x = B.rms_norm(h, self.norm, c.eps)
            h = B.add(h, B.mul_mat(w["down"], B.swiglu(B.mul_mat(w["gate"], x), B.mul_mat(w["up"], x))))
        return h

    def _logits(self, rows):
        return B.mul_mat(self.embed, B.rms_norm(rows.contiguous(), self.norm, self.cfg.eps))

    def prefill(self, prompts):
        """Packed prompts (lists of token ids) into the cache; the logits of their last tokens."""
        lens = [len(p) for p in prompts]
        for s, n in enumerate(lens):
            self.pages.grow(s, n)
        table = self.pages.table[:len(prompts)].cuda()
        dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
        ids = torch.tensor([t for p in prompts for t in p], dtype=torch.int32).cuda()
        pos = torch.cat([torch.arange(n, dtype=torch.int32) for n in lens]).cuda()
        h = self._forward(ids, pos, cu, dev_lens, table,
                          lambda n, q, k, v: B.flash_attn_packed(q, k, v, cu, status=self.status))
        return self._logits(h[(cu[1:] - 1).long()]), lens

    def step(self, tokens, lens):
        """One new token of each sequence (int32 on the device); their logits. `lens` counts it."""
        n = len(lens)
        for s, m in enumerate(lens):
            self.pages.grow(s, m)
        table = self.pages.table[:n].cuda()
        dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        h = self._forward(tokens, dev_lens - 1, cu, dev_lens, table,
                          lambda l, q, k, v: B.flash_attn_paged_batch(q, self.pages.k[l], self.pages.v[l], table, dev_lens,
                                                                      status=self.status))
        return self._logits(h)

    def generate(self, prompts, steps, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, seed=0):
        """`steps` tokens after each prompt: (prompts, steps) int32 on the host."""
        n = len(prompts)
        g = torch.Generator(device="cuda").manual_seed(seed)
        t = torch.full((n,), temperature, device="cuda")
        k = torch.full((n,), top_k, dtype=torch.int32, device="cuda")
        p, m = torch.full((n,), top_p, device="cuda"), torch.full((n,), min_p, device="cuda")
        logits, lens = self.prefill(prompts)
        out = []
        for _ in range(steps):
            tokens = B.sample(logits, torch.rand(n, device="cuda", generator=g), t, k, p, m, status=self.status)
            out.append(tokens)
            lens = [x + 1 for x in lens]
            logits = self.step(tokens, lens)
        for s in range(n):
            self.pages.release(s)
        if int(self.status):
            raise RuntimeError(f"device status {int(self.status)}")
        return torch.stack(out, 1).cpu()


def main():
    decoder = Decoder(Config())
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, decoder.cfg.vocab, (n,), generator=g).tolist() for n in (3, 150, 17, 64, 301)]
    for name, settings in (("greedy", {}), ("sampled", dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01))):
        tokens = decoder.generate(prompts, 8, **settings)
        for prompt, row in zip(prompts, tokens.tolist()):
            print(f"{name}: {len(prompt):4d} prompt tokens -> {row}")


if __name__ == "__main__":
    main()
