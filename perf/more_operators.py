"""Cases of what a server of many sequences needs besides the operators in operators.py: a
paged K/V cache held in 8 bits (append, read back, one-token attention over it),
one-token attention of batches whose sequences share a prefix, and the adjustment of
logits (penalties, biases, grammar masks) before a token is drawn.

``run`` computes a case either in plain torch operations (``own = False``) or through
the package's entry points (``own = True``). Shapes are those of the Qwen3 configurations
this repository runs (16 / 8 heads and 32 / 8 heads of 128, vocabulary 151936) and the
smaller head layouts its tests use. Sequence lengths are held as texts of comma-separated
numbers, so that a case is a dict of plain values.

The 8-bit cache: a row of head_dim elements (one token, one KV head) is x = q 2^e, with q in
e4m3 and e the least whole number with max |x| <= 448 2^e (at least -127), held as
an e8m0 number.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def _ints(text):
    return [int(x) for x in str(text).split(",")]


def _text(values):
    return ",".join(str(int(v)) for v in values)


# ---------------------------------------------------------------------------
# cases

def _append(name, dtype, heads, block, new, past):
    return {"name": name, "op": "append", "dtype": dtype, "Hkv": heads[1], "D": heads[2], "block": block,
            "new": _text(new), "past": _text(past)}


def _read(name, dtype, heads, block, rows, past):
    return {"name": name, "op": "read", "dtype": dtype, "Hkv": heads[1], "D": heads[2], "block": block,
            "rows": _text(rows), "past": _text(past)}


def _decode(name, dtype, heads, block, lens):
    return {"name": name, "op": "decode", "dtype": dtype, "Hq": heads[0], "Hkv": heads[1], "D": heads[2],
            "block": block, "lens": _text(lens)}


def _shared(name, dtype, heads, block, prefix, seqs, lens):
    """Group g: seqs[g] sequences behind a prefix of prefix[g] positions; lens: each sequence's own."""
    return {"name": name, "op": "shared", "dtype": dtype, "Hq": heads[0], "Hkv": heads[1], "D": heads[2],
            "block": block, "prefix": _text(prefix), "seqs": _text(seqs), "lens": _text(lens)}


def _logits(name, dtype, vocab, history, biases, mask):
    return {"name": name, "op": "logits", "dtype": dtype, "vocab": vocab, "history": _text(history), "biases": biases,
            "mask": mask}


def _spread(n, low, high, step):
    """n lengths over [low, high] in a fixed scattered order (ragged batches)."""
    return [low + (i * step) % (high - low + 1) for i in range(n)]


def listed():
    return [
        # one decode step's new rows of 64 users
        _append("q8_append_step64_bf16", "bf16", (32, 8, 128), 16, [1] * 64, _spread(64, 4, 4095, 1277)),
        # the rows of packed prompts into the cache
        _append("q8_append_prompts_f32", "f32", (16, 8, 128), 16, [1, 777, 64, 1333, 129, 2, 511, 250, 38, 991],
                [0, 0, 300, 0, 17, 1024, 0, 5, 0, 0]),
        # one short cached prompt read back, on the small test layout: latency
        _read("q8_read_one_f16", "f16", (8, 4, 64), 16, [301], [0]),
        # the cached heads of prompts that go on in chunks
        _read("q8_read_chunks_bf16", "bf16", (32, 8, 128), 16, [4096, 777, 8191, 64, 12000, 2, 5003, 2048], [0, 9, 0, 0, 0, 100, 3, 0]),
        # one user's step at a short context: latency
        _decode("q8_decode_one_f32", "f32", (16, 8, 128), 16, [301]),
        # a busy server: 64 users, contexts from a few tokens to 4k
        _decode("q8_decode_ragged64_bf16", "bf16", (32, 8, 128), 16, _spread(64, 5, 4096, 1277)),
        # F32 queries, long contexts, large pages
        _decode("q8_decode_long16_f32", "f32", (16, 8, 128), 128, _spread(16, 1500, 8192, 2903)),
        # a few users behind a short instruction
        _shared("shared_short_f32", "f32", (16, 8, 128), 16, [301], [4], [3, 40, 17, 90]),
        # 64 users behind one long document
        _shared("shared_64_bf16", "bf16", (32, 8, 128), 16, [8192], [64], _spread(64, 5, 1024, 389)),
        # several instructions at once, some users without any (an empty prefix)
        _shared("shared_groups_f16", "f16", (8, 4, 64), 16, [1000, 0, 3001, 131, 517], [20, 7, 11, 1, 3],
                _spread(42, 1, 600, 131)),
        # one user, everything on
        _logits("logits_one", "f32", 151936, [2000], 30, "mixed"),
        # a full batch
        _logits("logits_batch256", "f32", 151936, _spread(256, 0, 4000, 1511), 30, "mixed"),
    ]


_LAYOUTS = [(16, 8, 128), (32, 8, 128), (8, 4, 64), (4, 4, 64), (16, 2, 64), (16, 1, 128)]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _split(rng, total, parts):
    """`total` in `parts` uneven pieces, each at least one."""
    w = [rng.random() ** 3 + 1e-3 for _ in range(parts)]
    s = sum(w)
    return [max(1, int(total * x / s)) for x in w]


def draw(rng):
    op = rng.choice(["append", "read", "decode", "shared", "logits"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads = rng.choice(_LAYOUTS)
    block = rng.choice([8, 16, 32, 100, 128])
    if op == "append":
        if rng.random() < 0.5:
            new = [1] * _log_int(rng, 1, 128)
        else:
            total = _log_int(rng, 16, 4000)
            new = _split(rng, total, min(total, _log_int(rng, 1, 24)))
        c = _append("", dtype, heads, block, new, [rng.choice([0, _log_int(rng, 1, 1500)]) for _ in new])
    elif op == "read":
        total = _log_int(rng, 1, 16000 if dtype == "f32" else 32000)
        rows = _split(rng, total, min(total, _log_int(rng, 1, 24)))
        c = _read("", dtype, heads, block, rows, [rng.choice([0, 0, _log_int(rng, 1, 200)]) for _ in rows])
    elif op == "decode":
        n = _log_int(rng, 1, 96)
        high = min(8192, 200000 // n)
        c = _decode("", dtype, heads, block, [_log_int(rng, 1, high) for _ in range(n)])
    elif op == "shared":
        n = _log_int(rng, 1, 64)
        seqs = _split(rng, n, min(n, rng.randint(1, 5)))
        while sum(seqs) > 64:
            seqs[seqs.index(max(seqs))] -= 1
        prefix = [rng.choice([0, 1, 1, 1]) * _log_int(rng, 1, 8192 // len(seqs)) for _ in seqs]
        c = _shared("", dtype, heads, block, prefix, seqs, [rng.choice([0, 1, 1, 1]) * _log_int(rng, 1, 1024) for _ in range(sum(seqs))])
    else:
        n = _log_int(rng, 1, 192)
        vocab = rng.choice([512, 32003, _log_int(rng, 300, 151936), 151936])
        c = _logits("", dtype, vocab, [rng.choice([0, _log_int(rng, 1, 4000)]) for _ in range(n)], rng.choice([0, 1, 30]),
                    rng.choice(["none", "mixed", "sparse"]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _cumulative(lens):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens, dtype=torch.int32).cumsum(0)
    return t.cuda()


def _lengths(lens):
    return torch.tensor(lens, dtype=torch.int32).cuda()


def _pages(lens, block, g, spare=7):
    """A block table over a pool in shuffled order, with some spare blocks."""
    per = [-(-n // block) for n in lens]
    blocks = sum(per) + spare
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros((len(lens), max(1, max(per))), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    return table, blocks, at, order


def _quantise(x):
    """Rows (last axis) as e4m3 elements and e8m0 scales."""
    x = x.float()
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e with m in [1/2, 1): 448 = 7/8 2^9
    e = e - 9 + (m > 0.875)
    e = torch.where(top == 0, torch.full_like(e, -127), e).clamp(min=-127)
    q = torch.ldexp(x, -e[..., None]).to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _keys(shape, g):
    """Key rows: some columns of a head are much larger than others, as behind a rotation."""
    return torch.randn(shape, device="cuda", generator=g) * torch.exp(0.6 * torch.randn(shape[-2:], device="cuda", generator=g))


def _values(shape, g):
    """Value rows: tokens differ in magnitude."""
    return torch.randn(shape, device="cuda", generator=g) * torch.exp(0.5 * torch.randn(shape[:-1], device="cuda", generator=g))[..., None]


def _pool8(s, blocks, case, g):
    """An 8-bit cache in use: every block holds rows. Scales are (blocks, Hkv, block_tokens)."""
    shape = (blocks, case["block"], case["Hkv"], case["D"])
    for name, make in (("k", _keys), ("v", _values)):
        q, e = _quantise(make(shape, g))
        s[name + "_pool"] = q
        s[name + "_scale"] = e.view(torch.uint8).transpose(1, 2).contiguous().view(torch.float8_e8m0fnu)


def _mask_words(allowed):
    """(n, vocab) truth values as 32-bit words, token t in bit t % 32 of word t / 32."""
    n, vocab = allowed.shape
    pad = torch.zeros((n, -vocab % 32), dtype=torch.bool, device=allowed.device)
    bits = torch.cat([allowed, pad], 1).view(n, -1, 32)
    words = (bits.long() << torch.arange(32, device=allowed.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]
    s = {"op": op, "dtype": dtype}

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(dtype)

    if op in ("append", "read"):
        new, past = _ints(case["new" if op == "append" else "rows"]), _ints(case["past"])
        lens = [a + b for a, b in zip(new, past)]
        s["table"], blocks, _, _ = _pages(lens, case["block"], g)
        _pool8(s, blocks, case, g)
        s["cu"], s["lens"], s["total"] = _cumulative(new), _lengths(lens), sum(new)
        if op == "append":
            s["k"] = _keys((sum(new), case["Hkv"], case["D"]), g).to(dtype)
            s["v"] = _values((sum(new), case["Hkv"], case["D"]), g).to(dtype)
    elif op == "decode":
        lens = _ints(case["lens"])
        s["table"], blocks, _, _ = _pages(lens, case["block"], g)
        _pool8(s, blocks, case, g)
        s["q"], s["lens"] = normal(len(lens), case["Hq"], case["D"]), _lengths(lens)
    elif op == "shared":
        lens, prefix, seqs = _ints(case["lens"]), _ints(case["prefix"]), _ints(case["seqs"])
        both, blocks, _, _ = _pages(prefix + lens, case["block"], g)
        wide = [max(1, max(-(-n // case["block"]) for n in part)) for part in (prefix, lens)]
        s["prefix_table"] = both[:len(prefix), :wide[0]].contiguous()
        s["table"] = both[len(prefix):, :wide[1]].contiguous()
        s["q"] = normal(len(lens), case["Hq"], case["D"])
        shape = (blocks, case["block"], case["Hkv"], case["D"])
        s["k_pool"], s["v_pool"] = _keys(shape, g).to(dtype), _values(shape, g).to(dtype)
        s["prefix_lens"], s["lens"], s["cu_seqs"] = _lengths(prefix), _lengths(lens), _cumulative(seqs)
    else:
        history, vocab = _ints(case["history"]), case["vocab"]
        n = len(history)
        # a language model's logits: a broad bulk and a few dozen likely tokens
        x = torch.randn((n, vocab), device="cuda", generator=g) * 2.0
        hot = torch.randint(0, vocab, (n, 40), device="cuda", generator=g)
        x.scatter_add_(1, hot, torch.rand((n, 40), device="cuda", generator=g) * 10.0)
        s["logits"] = x.to(dtype)
        # text repeats its frequent tokens
        u = torch.rand(sum(history), device="cuda", generator=g)
        s["tokens"] = (u ** 4 * vocab).to(torch.int32).clamp(max=vocab - 1)
        s["cu_tokens"] = _cumulative(history)
        s["prompt_lens"] = (torch.rand(n, device="cuda", generator=g) * _lengths(history)).to(torch.int32)

        def pick(values):
            at = torch.randint(0, len(values), (n,), device="cuda", generator=g)
            return torch.tensor(values, dtype=torch.float32).cuda()[at]

        s["repetition"], s["frequency"], s["presence"] = pick([1.0, 1.05, 1.3]), pick([0.0, 0.2, -0.1]), pick([0.0, 0.5])
        if case["biases"]:  # different tokens of a row
            step = max(1, vocab // case["biases"])
            ids = torch.arange(case["biases"], device="cuda")[None] * step + torch.randint(0, step, (n, case["biases"]), device="cuda", generator=g)
            s["bias_ids"] = ids.clamp(max=vocab - 1).to(torch.int32).view(-1)
            s["bias_values"] = torch.randn(n * case["biases"], device="cuda", generator=g) * 5.0
            s["cu_bias"] = _cumulative([case["biases"]] * n)
        if case["mask"] != "none":
            keep = pick([1.0, 0.5, 0.01] if case["mask"] == "mixed" else [0.0, 0.001, 0.01])
            s["mask"] = _mask_words(torch.rand((n, vocab), device="cuda", generator=g) < keep[:, None])
    return s


# ---------------------------------------------------------------------------
# one pass

def _package():
    here = os.path.join(os.getcwd(), "infer-llm_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import b200infer
    return b200infer


_B = None


def run(state):
    global _B
    op, s = state["op"], state
    if own:
        if _B is None:
            _B = _package()
        if op == "append":
            _B.paged_kv_append_q8(s["k"], s["v"], s["cu"], s["lens"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"])
            return s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"]
        if op == "read":
            return _B.paged_kv_read_q8(s["cu"], s["lens"], s["total"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"],
                                       s["table"], dtype=s["dtype"])
        if op == "decode":
            return _B.flash_attn_paged_batch_q8(s["q"], s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"], s["table"], s["lens"])
        if op == "shared":
            return _B.flash_attn_paged_shared(s["q"], s["k_pool"], s["v_pool"], s["prefix_table"], s["prefix_lens"], s["cu_seqs"],
                                              s["table"], s["lens"])
        return _B.adjust_logits(s["logits"], s["tokens"], s["cu_tokens"], s["prompt_lens"], s["repetition"], s["frequency"],
                                s["presence"], s.get("bias_ids"), s.get("bias_values"), s.get("cu_bias"), s.get("mask"))
    return _PLAIN[op](s)


def _rows_of(s, cu):
    """The page and the place in it of each packed row: a sequence's rows are its last positions."""
    t = torch.arange(s["total"], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = s["lens"].long()[b] - cu[b + 1] + t
    block = s["k_pool"].shape[1]
    return s["table"].long()[b, pos // block], pos % block


def _plain_append(s):
    page, place = _rows_of(s, s["cu"].long())
    for name in ("k", "v"):
        q, e = _quantise(s[name])
        s[name + "_pool"].view(torch.uint8)[page, place] = q.view(torch.uint8)
        s[name + "_scale"].view(torch.uint8)[page, :, place] = e.view(torch.uint8)
    return s["k_pool"], s["v_pool"], s["k_scale"], s["v_scale"]


def _plain_read(s):
    page, place = _rows_of(s, s["cu"].long())
    out = []
    for name in ("k", "v"):
        q = s[name + "_pool"].view(torch.uint8)[page, place].view(torch.float8_e4m3fn).float()
        e = s[name + "_scale"].view(torch.uint8)[page, :, place].view(torch.float8_e8m0fnu).float()
        out.append((q * e[..., None]).to(s["dtype"]))
    return tuple(out)


def _softmax(scores, seen):
    """Softmax over the last axis of the entries that `seen` marks; a row with none is zero."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _places(table, block):
    """The pages of a padded batch's positions, and their places in them."""
    j = torch.arange(table.shape[1] * block, device=table.device)
    return j, table.long()[:, j // block], (j % block).expand(table.shape[0], -1)


def _plain_decode(s):
    """The pages gathered into one padded batch of F32 rows, then masked attention of one row each."""
    q, lens = s["q"].float(), s["lens"].long()
    B, Hq, D = q.shape
    block, Hkv = s["k_pool"].shape[1], s["k_pool"].shape[2]
    j, page, place = _places(s["table"], block)

    def rows(name):  # (B, Hkv, keys, D)
        x = s[name + "_pool"].view(torch.uint8)[page, place].view(torch.float8_e4m3fn).float()
        e = s[name + "_scale"].view(torch.uint8)[page, :, place].view(torch.float8_e8m0fnu).float()
        return (x * e[..., None]).permute(0, 2, 1, 3)

    qh = q.view(B, Hkv, Hq // Hkv, D)
    seen = (j[None, :] < lens[:, None])[:, None, None, :]
    p = _softmax(torch.matmul(qh, rows("k").transpose(-1, -2)) / math.sqrt(D), seen)
    return torch.matmul(p, rows("v")).reshape(B, Hq, D).to(s["q"].dtype)


def _plain_shared(s):
    """Every row against all prefixes (its own marked) and against its own pages."""
    q, lens, cu = s["q"].float(), s["lens"].long(), s["cu_seqs"].long()
    B, Hq, D = q.shape
    block, Hkv = s["k_pool"].shape[1], s["k_pool"].shape[2]
    G, groups = Hq // Hkv, cu.shape[0] - 1
    j, page, place = _places(s["table"], block)
    kh, vh = (s[name][page, place].float().permute(0, 2, 1, 3) for name in ("k_pool", "v_pool"))  # (B, Hkv, keys, D)
    i, ppage, pplace = _places(s["prefix_table"], block)
    pk, pv = (s[name][ppage, pplace].float().reshape(-1, Hkv, D).permute(1, 0, 2) for name in ("k_pool", "v_pool"))  # (Hkv, all, D)
    group = torch.searchsorted(cu, torch.arange(B, device=q.device), right=True) - 1
    seen_own = j[None, :] < lens[:, None]
    seen_prefix = (group[:, None, None] == torch.arange(groups, device=q.device)[None, :, None]) & \
        (i[None, None, :] < s["prefix_lens"].long()[None, :, None])
    qh = q.view(B, Hkv, G, D)
    own_scores = torch.matmul(qh, kh.transpose(-1, -2))
    qp = qh.permute(1, 0, 2, 3).reshape(Hkv, B * G, D)
    prefix_scores = torch.matmul(qp, pk.transpose(-1, -2)).view(Hkv, B, G, -1).permute(1, 0, 2, 3)
    scores = torch.cat([prefix_scores, own_scores], -1) / math.sqrt(D)
    p = _softmax(scores, torch.cat([seen_prefix.view(B, -1), seen_own], 1)[:, None, None, :])
    n = pk.shape[1]
    from_prefix = torch.matmul(p[..., :n].permute(1, 0, 2, 3).reshape(Hkv, B * G, n), pv).view(Hkv, B, G, D).permute(1, 0, 2, 3)
    return (from_prefix + torch.matmul(p[..., n:], vh)).reshape(B, Hq, D).to(s["q"].dtype)


def _plain_logits(s):
    """Repetition, then frequency and presence, then bias, then the mask."""
    x = s["logits"].float()
    n, vocab = x.shape
    cu = s["cu_tokens"].long()
    t = torch.arange(s["tokens"].shape[0], device=x.device)
    row = torch.searchsorted(cu, t, right=True) - 1
    at = row * vocab + s["tokens"].long()
    drawn = t - cu[row] >= s["prompt_lens"].long()[row]  # not of the prompt
    counts = torch.zeros(n * vocab, device=x.device).index_add_(0, at, drawn.float()).view(n, vocab)
    known = torch.zeros(n * vocab, dtype=torch.bool, device=x.device).index_fill_(0, at, True).view(n, vocab)
    r = s["repetition"][:, None]
    x = torch.where(known, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * counts - s["presence"][:, None] * (counts > 0)
    if "bias_ids" in s:
        m = torch.arange(s["bias_ids"].shape[0], device=x.device)
        row = torch.searchsorted(s["cu_bias"].long(), m, right=True) - 1
        x.view(-1).index_add_(0, row * vocab + s["bias_ids"].long(), s["bias_values"])
    if "mask" in s:
        j = torch.arange(vocab, device=x.device)
        allowed = (s["mask"][:, j // 32] >> (j % 32)) & 1
        x = torch.where(allowed != 0, x, torch.full_like(x, -math.inf))
    return x.to(s["logits"].dtype)


_PLAIN = {"append": _plain_append, "read": _plain_read, "decode": _plain_decode, "shared": _plain_shared, "logits": _plain_logits}


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    op, e = case["op"], _BYTES[case["dtype"]]
    if op in ("append", "read"):
        rows = sum(_ints(case["new" if op == "append" else "rows"])) * case["Hkv"] * 2
        return {"bytes": rows * (case["D"] * (e + 1) + 1), "flops": rows * case["D"]}
    if op == "decode":
        lens = _ints(case["lens"])
        return {"bytes": 2 * sum(lens) * case["Hkv"] * (case["D"] + 1) + 2 * e * len(lens) * case["Hq"] * case["D"],
                "flops": 4 * case["Hq"] * case["D"] * sum(lens)}
    if op == "shared":
        lens, prefix, seqs = _ints(case["lens"]), _ints(case["prefix"]), _ints(case["seqs"])
        return {"bytes": e * case["D"] * (2 * (sum(lens) + sum(prefix)) * case["Hkv"] + 2 * len(lens) * case["Hq"]),
                "flops": 4 * case["Hq"] * case["D"] * (sum(lens) + sum(a * b for a, b in zip(prefix, seqs)))}
    history = _ints(case["history"])
    n, vocab = len(history), case["vocab"]
    masks = 0 if case["mask"] == "none" else n * -(-vocab // 32) * 4
    return {"bytes": 2 * e * n * vocab + masks + 4 * sum(history) + 8 * n * case["biases"], "flops": n * vocab}


# ---------------------------------------------------------------------------
# the definition in 64 bits

def _e4m3_exact(x):
    """Rows (last axis) in 64 bits: elements rounded to four binary digits (no finer than 2^-9), and scales."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448.0))  # whole but for the logarithm's rounding
    e = torch.where(448.0 * torch.exp2(e - 1) >= top, e - 1, e)
    e = torch.where(448.0 * torch.exp2(e) < top, e + 1, e)
    e = torch.where(top == 0, torch.full_like(e, -127.0), e).clamp(min=-127.0)
    y = x / torch.exp2(e)
    place = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(place.clamp(min=-6.0) - 3.0)
    return torch.round(y / step) * step, torch.exp2(e[..., 0])  # (torch.round: ties to even)


def _held64(pool, scale, blocks, n):
    """The first n positions of a list of blocks, (n, Hkv, D)."""
    x = pool.view(torch.uint8)[blocks].view(torch.float8_e4m3fn).double()
    e = scale.view(torch.uint8)[blocks].view(torch.float8_e8m0fnu).double()
    return (x * e.transpose(1, 2)[..., None]).flatten(0, 1)[:n]


def _one_row64(q, k, v):
    """q (Hq, D) over k, v (m, Hkv, D)."""
    Hq, D = q.shape
    if k.shape[0] == 0:
        return torch.zeros((Hq, D), dtype=torch.float64, device=q.device)
    rep = Hq // k.shape[1]
    kk, vv = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    a = torch.einsum("hd,mhd->hm", q.double(), kk) / D ** 0.5
    return torch.einsum("hm,mhd->hd", torch.softmax(a, -1), vv)


def exact(case, seed):
    op = case["op"]
    s = prepare(case, seed)
    if op == "logits":
        return _logits64(s)
    block = case["block"]
    table = s["table"].long()

    def pages(row, n):
        return row[:-(-n // block)]

    if op == "decode":
        return torch.stack([_one_row64(s["q"][b], *(_held64(s[x + "_pool"], s[x + "_scale"], pages(table[b], n), n) for x in "kv"))
                            for b, n in enumerate(_ints(case["lens"]))])
    if op == "shared":
        out, b, lens = [], 0, _ints(case["lens"])
        for g, (prefix, count) in enumerate(zip(_ints(case["prefix"]), _ints(case["seqs"]))):
            head = [s[x][pages(s["prefix_table"][g].long(), prefix)].flatten(0, 1)[:prefix] for x in ("k_pool", "v_pool")]
            for _ in range(count):
                tail = [s[x][pages(table[b], lens[b])].flatten(0, 1)[:lens[b]] for x in ("k_pool", "v_pool")]
                out.append(_one_row64(s["q"][b], torch.cat([head[0], tail[0]]), torch.cat([head[1], tail[1]])))
                b += 1
        return torch.stack(out)
    lens = s["lens"].tolist()
    counts = _ints(case["new" if op == "append" else "rows"])
    if op == "read":
        return tuple(torch.cat([_held64(s[x + "_pool"], s[x + "_scale"], pages(table[b], n), n)[n - counts[b]:]
                                for b, n in enumerate(lens)]) for x in "kv")
    held = {x: s[x + "_pool"].double() for x in "kv"}
    scales = {x: s[x + "_scale"].double() for x in "kv"}
    at = 0
    for b, (n, m) in enumerate(zip(lens, counts)):
        pos = torch.arange(n - m, n, device="cuda")
        page, place = table[b][pos // block], pos % block
        for x in "kv":
            q, e = _e4m3_exact(s[x][at:at + m].double())
            held[x][page, place] = q
            scales[x][page, :, place] = e
        at += m
    return held["k"], held["v"], scales["k"], scales["v"]


def _logits64(s):
    x = s["logits"].double()
    vocab = x.shape[1]
    cu, cb = s["cu_tokens"].tolist(), s["cu_bias"].tolist() if "cu_bias" in s else None
    split = s["prompt_lens"].tolist()
    r, f, p = (s[name].double() for name in ("repetition", "frequency", "presence"))
    for b in range(x.shape[0]):  # row by row, the tokens that occur
        ids = s["tokens"][cu[b]:cu[b + 1]].long()
        some = torch.unique(ids)
        y = x[b, some]
        x[b, some] = torch.where(y > 0, y / r[b], y * r[b])
        ids, times = torch.unique(ids[split[b]:], return_counts=True)
        x[b, ids] -= f[b] * times + p[b]
        if cb is not None:
            ids = s["bias_ids"][cb[b]:cb[b + 1]].long()
            x[b, ids] += s["bias_values"][cb[b]:cb[b + 1]].double()
        if "mask" in s:
            words = s["mask"][b].long() & 0xFFFFFFFF
            bits = ((words[:, None] >> torch.arange(32, device=words.device)) & 1).view(-1)[:vocab]
            x[b, bits == 0] = -math.inf
    return x
