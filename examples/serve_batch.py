"""Many sequences at once: prompts of different lengths are packed and prefilled together,
their K / V go into one paged cache, and every decode step attends, samples and appends for
all of them.

A Qwen3-shaped decoder with random weights on the single ops of the package (F32); with a
GPU: ``python examples/serve_batch.py``. ``Decoder.prefill`` and ``Decoder.step`` show how
flash_attn_packed, paged_kv_append, flash_attn_paged_batch and sample go together;
``cache="q8"`` holds the cache in 8 bits (paged_kv_append_q8, flash_attn_paged_batch_q8,
paged_kv_read_q8 where prompts go on in ``Decoder.extend``); a ``Prefix`` is prefilled once for
all sequences that begin with it (flash_attn_paged_shared); ``Decoder.generate`` takes
penalties, biases and allowed tokens (adjust_logits).
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

    def __init__(self, cfg, n_blocks, block_tokens, max_seqs, eight_bit=False):
        self.bt = block_tokens
        self.free = list(range(n_blocks))[::-1]
        shape = (cfg.layers, n_blocks, block_tokens, cfg.heads_kv, cfg.dim)
        kind = torch.float8_e4m3fn if eight_bit else torch.float32
        self.k = torch.empty(shape, device="cuda", dtype=kind)
        self.v = torch.empty(shape, device="cuda", dtype=kind)
        if eight_bit:  # one scale a token and KV head, a head's scales next to each other
            shape = (cfg.layers, n_blocks, cfg.heads_kv, block_tokens)
            self.k_scale = torch.empty(shape, device="cuda", dtype=torch.float8_e8m0fnu)
            self.v_scale = torch.empty(shape, device="cuda", dtype=torch.float8_e8m0fnu)
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


class Prefix:
    """Tokens that several sequences begin with: their blocks, held until `release`."""

    def __init__(self, pages, tokens):
        self.pages, self.tokens = pages, list(tokens)
        self.blocks = [pages.free.pop() for _ in range(-(-len(self.tokens) // pages.bt))]
        self.table = torch.tensor([self.blocks], dtype=torch.int32).cuda()
        self.lens = torch.tensor([len(self.tokens)], dtype=torch.int32).cuda()

    def release(self):
        self.pages.free += self.blocks
        self.blocks = []


class Decoder:
    def __init__(self, cfg, seed=0, n_blocks=512, block_tokens=16, max_seqs=16, cache="f32"):
        self.cfg, self.eight_bit = cfg, cache == "q8"
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
        self.pages = PagePool(cfg, n_blocks, block_tokens, max_seqs, self.eight_bit)
        self.status = torch.zeros(1, dtype=torch.int32, device="cuda")

    def _cache(self, layer):
        p = self.pages
        return (p.k[layer], p.v[layer]) + ((p.k_scale[layer], p.v_scale[layer]) if self.eight_bit else ())

    def _forward(self, ids, pos, cu_new, lens, table, attend):
        """Hidden rows of packed new tokens; `attend(layer, q, k, v)` is their attention."""
        c, h = self.cfg, B.get_rows(self.embed, ids)
        append = B.paged_kv_append_q8 if self.eight_bit else B.paged_kv_append
        T = ids.numel()
        for n, w in enumerate(self.layers):
            x = B.rms_norm(h, self.norm, c.eps)
            q = B.mul_mat(w["q"], x).view(T, c.heads, c.dim)
            k = B.mul_mat(w["k"], x).view(T, c.heads_kv, c.dim)
            v = B.mul_mat(w["v"], x).view(T, c.heads_kv, c.dim)
            q, k, _ = B.qk_norm_rope(q, k, self.head_norm, self.head_norm, self.freq, pos, c.eps, c.ctx)
            append(k, v, cu_new, lens, *self._cache(n), table, status=self.status)
            h = B.add(h, B.mul_mat(w["o"], attend(n, q, k, v).view(T, -1)))
            x = B.rms_norm(h, self.norm, c.eps)
            h = B.add(h, B.mul_mat(w["down"], B.swiglu(B.mul_mat(w["gate"], x), B.mul_mat(w["up"], x))))
        return h

    def _logits(self, rows):
        return B.mul_mat(self.embed, B.rms_norm(rows.contiguous(), self.norm, self.cfg.eps))

    def _held(self, layer, table, lens):
        """All cached K and V rows of each sequence, packed."""
        if self.eight_bit:
            cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
            return B.paged_kv_read_q8(cu, torch.tensor(lens, dtype=torch.int32).cuda(), sum(lens), *self._cache(layer), table,
                                      dtype=torch.float32, status=self.status)
        return tuple(torch.cat([pool[row.long()].flatten(0, 1)[:n] if n else pool[0, :0] for row, n in zip(table, lens)])
                     for pool in self._cache(layer))

    def extend(self, chunks, past, prefix=None):
        """The next tokens of each sequence (lists of ids, packed) behind the past[s] it has cached, and behind
        the prefix; the logits of their last tokens, and the new lengths."""
        new = [len(p) for p in chunks]
        lens = [a + b for a, b in zip(new, past)]
        for s, n in enumerate(lens):
            self.pages.grow(s, n)
        table = self.pages.table[:len(chunks)].cuda()
        head = len(prefix.tokens) if prefix else 0
        cu = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
        keys = torch.tensor([0] + [head + n for n in lens], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
        ids = torch.tensor([t for p in chunks for t in p], dtype=torch.int32).cuda()
        pos = torch.cat([torch.arange(head + p, head + n, dtype=torch.int32) for p, n in zip(past, lens)]).cuda()

        def attend(n, q, k, v):
            if not head and not any(past):
                return B.flash_attn_packed(q, k, v, cu, status=self.status)
            own = [torch.split(x, lens) for x in self._held(n, table, lens)]
            if head:
                own = [[torch.cat([x, y]) for y in ys] for x, ys in zip(self._held(n, prefix.table, [head]), own)]
            return B.flash_attn_packed(q, torch.cat(list(own[0])), torch.cat(list(own[1])), cu, keys, status=self.status)

        h = self._forward(ids, pos, cu, torch.tensor(lens, dtype=torch.int32).cuda(), table, attend)
        return self._logits(h[(cu[1:] - 1).long()]), lens

    def prefill(self, prompts, prefix=None):
        """Packed prompts (lists of token ids) into the cache; the logits of their last tokens."""
        return self.extend(prompts, [0] * len(prompts), prefix)

    def prefix(self, tokens):
        """Common first tokens of later prompts, prefilled once."""
        p = Prefix(self.pages, tokens)
        n = len(p.tokens)
        ids, pos = torch.tensor(p.tokens, dtype=torch.int32).cuda(), torch.arange(n, dtype=torch.int32).cuda()
        cu = torch.tensor([0, n], dtype=torch.int32).cuda()
        self._forward(ids, pos, cu, p.lens, p.table, lambda l, q, k, v: B.flash_attn_packed(q, k, v, cu, status=self.status))
        return p

    def step(self, tokens, lens, prefix=None):
        """One new token of each sequence (int32 on the device); their logits. `lens` counts it, not the prefix."""
        n = len(lens)
        for s, m in enumerate(lens):
            self.pages.grow(s, m)
        table = self.pages.table[:n].cuda()
        dev_lens = torch.tensor(lens, dtype=torch.int32).cuda()
        cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        head = len(prefix.tokens) if prefix else 0
        if self.eight_bit and prefix:
            raise ValueError("a shared prefix takes an F32 cache")
        group = torch.tensor([0, n], dtype=torch.int32).cuda()

        def attend(l, q, k, v):
            if prefix:
                return B.flash_attn_paged_shared(q, *self._cache(l), prefix.table, prefix.lens, group, table, dev_lens,
                                                 status=self.status)
            batch = B.flash_attn_paged_batch_q8 if self.eight_bit else B.flash_attn_paged_batch
            return batch(q, *self._cache(l), table, dev_lens, status=self.status)

        return self._logits(self._forward(tokens, dev_lens - 1 + head, cu, dev_lens, table, attend))

    def generate(self, prompts, steps, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, seed=0, prefix=None,
                 repetition=1.0, frequency=0.0, presence=0.0, bias=None, allowed=None):
        """`steps` tokens after each prompt: (prompts, steps) int32 on the host. bias: {token: number}, allowed: (vocab)
        truth values, for all sequences."""
        n = len(prompts)
        g = torch.Generator(device="cuda").manual_seed(seed)

        def each(x, kind=torch.float32):
            return torch.full((n,), x, dtype=kind, device="cuda")

        t, k, p, m = each(temperature), each(top_k, torch.int32), each(top_p), each(min_p)
        history = [torch.tensor((prefix.tokens if prefix else []) + list(x), dtype=torch.int32).cuda() for x in prompts]
        begin = torch.tensor([len(x) for x in history], dtype=torch.int32).cuda()
        ask = {}
        if repetition != 1.0 or frequency or presence:
            ask.update(prompt_lens=begin, repetition=each(repetition), frequency=each(frequency), presence=each(presence))
        if bias:
            ask.update(bias_ids=torch.tensor(list(bias) * n, dtype=torch.int32).cuda(),
                       bias_values=torch.tensor(list(bias.values()) * n, dtype=torch.float32).cuda(),
                       cu_bias=torch.arange(n + 1, dtype=torch.int32, device="cuda") * len(bias))
        if allowed is not None:
            bits = torch.nn.functional.pad(allowed.cuda(), (0, -allowed.numel() % 32)).view(-1, 32).long()
            words = (bits << torch.arange(32, device="cuda")).sum(1)
            ask["mask"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).int().expand(n, -1)
        logits, lens = self.prefill(prompts, prefix)
        out = []
        for _ in range(steps):
            if ask:
                if "repetition" in ask:
                    ask["tokens"] = torch.cat(history)
                    ask["cu_tokens"] = torch.tensor([0] + [x.numel() for x in history], dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
                logits = B.adjust_logits(logits, **ask, out=logits, status=self.status)
            tokens = B.sample(logits, torch.rand(n, device="cuda", generator=g), t, k, p, m, status=self.status)
            out.append(tokens)
            history = [torch.cat([x, tokens[s:s + 1]]) for s, x in enumerate(history)]
            lens = [x + 1 for x in lens]
            logits = self.step(tokens, lens, prefix)
        for s in range(n):
            self.pages.release(s)
        if int(self.status):
            raise RuntimeError(f"device status {int(self.status)}")
        return torch.stack(out, 1).cpu()


def main():
    decoder = Decoder(Config())
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, decoder.cfg.vocab, (n,), generator=g).tolist() for n in (3, 150, 17, 64, 301)]
    small = Decoder(Config(), cache="q8")
    instruction = decoder.prefix(torch.randint(0, decoder.cfg.vocab, (100,), generator=g).tolist())
    sampled = dict(temperature=0.8, top_k=50, top_p=0.95, min_p=0.01)
    for name, d, settings in (("greedy", decoder, {}), ("sampled", decoder, sampled), ("8-bit cache", small, {}),
                              ("behind a prefix", decoder, dict(prefix=instruction)),
                              ("penalised", decoder, dict(repetition=1.3, presence=0.5, bias={7: -100.0}, **sampled))):
        tokens = d.generate(prompts, 8, **settings)
        for prompt, row in zip(prompts, tokens.tolist()):
            print(f"{name}: {len(prompt):4d} prompt tokens -> {row}")


if __name__ == "__main__":
    main()
