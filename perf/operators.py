"""Cases of the batched-serving operators: packed causal prefill attention, append to a
paged K/V cache, one-token attention over that cache, and token sampling.

``run`` computes a case either in plain torch operations (``own = False``) or through
the package's entry points (``own = True``). Shapes are those of the Qwen3 configurations
this repository runs (16 / 8 heads and 32 / 8 heads of 128, vocabulary 151936) and the
smaller head layouts its tests use. Sequence lengths are held as texts of comma-separated
numbers, so that a case is a dict of plain values.
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

def _prefill(name, dtype, heads, q_lens, past=None):
    past = [0] * len(q_lens) if past is None else past
    return {"name": name, "op": "prefill", "dtype": dtype, "Hq": heads[0], "Hkv": heads[1], "D": heads[2],
            "q_lens": _text(q_lens), "past": _text(past)}


def _append(name, dtype, heads, block, new, past):
    return {"name": name, "op": "append", "dtype": dtype, "Hkv": heads[1], "D": heads[2], "block": block,
            "new": _text(new), "past": _text(past)}


def _decode(name, dtype, heads, block, lens):
    return {"name": name, "op": "decode", "dtype": dtype, "Hq": heads[0], "Hkv": heads[1], "D": heads[2],
            "block": block, "lens": _text(lens)}


def _sample(name, dtype, rows, vocab, mode):
    return {"name": name, "op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "mode": mode}


def _spread(n, low, high, step):
    """n lengths over [low, high] in a fixed scattered order (ragged batches)."""
    return [low + (i * step) % (high - low + 1) for i in range(n)]


def listed():
    return [
        # one short user prompt on the small test layout: latency is all there is
        _prefill("prefill_short_f32", "f32", (8, 4, 64), [37]),
        # the repository's long-prompt configuration (2048 tokens, 16 / 8 heads, exact F32)
        _prefill("prefill_2048_f32", "f32", (16, 8, 128), [2048]),
        # an admission step of a server: prompts of very different lengths packed together
        _prefill("prefill_packed_bf16", "bf16", (16, 8, 128),
                 [1, 777, 64, 1333, 129, 2, 511, 250, 38, 991]),
        # the tail chunks of prompts whose heads are already cached (keys longer than queries)
        _prefill("prefill_chunk_f16", "f16", (8, 4, 64), [256, 511, 97], [1024, 3001, 5]),
        # the largest: one long document on the 32 / 8 head layout
        _prefill("prefill_8192_bf16", "bf16", (32, 8, 128), [8192]),
        # one user's step at a short context: latency
        _decode("decode_one_f32", "f32", (16, 8, 128), 16, [301]),
        # a busy server: 64 users, contexts from a few tokens to 4k
        _decode("decode_ragged64_bf16", "bf16", (32, 8, 128), 16, _spread(64, 5, 4096, 1277)),
        # F32 caches, long contexts, large pages
        _decode("decode_long16_f32", "f32", (16, 8, 128), 128, _spread(16, 1500, 8192, 2903)),
        # one decode step's new rows of 64 users
        _append("append_step64_bf16", "bf16", (32, 8, 128), 16, [1] * 64, _spread(64, 4, 4095, 1277)),
        # the rows of packed prompts into the cache
        _append("append_prompts_f32", "f32", (16, 8, 128), 16, [1, 777, 64, 1333, 129, 2, 511, 250, 38, 991],
                [0, 0, 300, 0, 17, 1024, 0, 5, 0, 0]),
        # one user, every filter on
        _sample("sample_one", "f32", 1, 151936, "filters"),
        # a full batch with mixed settings
        _sample("sample_batch256", "f32", 256, 151936, "mixed"),
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
    op = rng.choice(["prefill", "decode", "append", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    heads = rng.choice(_LAYOUTS)
    if op == "prefill":
        total = _log_int(rng, 16, 6000)
        q_lens = _split(rng, total, min(total, _log_int(rng, 1, 24)))
        past = [rng.choice([0, 0, _log_int(rng, 1, 1000)]) for _ in q_lens]
        while sum(past) > 4000:
            past = [p // 2 for p in past]
        c = _prefill("", dtype, heads, q_lens, past)
    elif op == "decode":
        n = _log_int(rng, 1, 96)
        high = min(8192, 200000 // n)
        c = _decode("", dtype, heads, rng.choice([8, 16, 32, 100, 128]), [_log_int(rng, 1, high) for _ in range(n)])
    elif op == "append":
        if rng.random() < 0.5:
            new = [1] * _log_int(rng, 1, 128)
        else:
            total = _log_int(rng, 16, 4096)
            new = _split(rng, total, min(total, _log_int(rng, 1, 24)))
        c = _append("", dtype, heads, rng.choice([8, 16, 32, 100, 128]), new, [rng.choice([0, _log_int(rng, 1, 1500)]) for _ in new])
    else:
        c = _sample("", dtype, _log_int(rng, 1, 192), rng.choice([512, 32003, _log_int(rng, 300, 151936), 151936]),
                    rng.choice(["filters", "mixed", "temperature"]))
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


def _pages(lens, block, g):
    """A block table over a pool in shuffled order, with some spare blocks."""
    per = [-(-n // block) for n in lens]
    blocks = sum(per) + 7
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    table = torch.zeros((len(lens), max(per)), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    return table, blocks


def prepare(case, seed):
    g = _gen(seed)
    op, dtype = case["op"], _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(dtype)

    s = {"op": op}
    if op == "prefill":
        ql, past = _ints(case["q_lens"]), _ints(case["past"])
        kl = [a + b for a, b in zip(ql, past)]
        s["q"] = normal(sum(ql), case["Hq"], case["D"])
        s["k"] = normal(sum(kl), case["Hkv"], case["D"])
        s["v"] = normal(sum(kl), case["Hkv"], case["D"])
        s["cu_q"], s["cu_k"] = _cumulative(ql), _cumulative(kl)
    elif op == "decode":
        lens = _ints(case["lens"])
        s["table"], blocks = _pages(lens, case["block"], g)
        s["q"] = normal(len(lens), case["Hq"], case["D"])
        s["k_pool"] = normal(blocks, case["block"], case["Hkv"], case["D"])
        s["v_pool"] = normal(blocks, case["block"], case["Hkv"], case["D"])
        s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    elif op == "append":
        new, past = _ints(case["new"]), _ints(case["past"])
        lens = [a + b for a, b in zip(new, past)]
        s["table"], blocks = _pages(lens, case["block"], g)
        s["k"] = normal(sum(new), case["Hkv"], case["D"])
        s["v"] = normal(sum(new), case["Hkv"], case["D"])
        s["k_pool"] = normal(blocks, case["block"], case["Hkv"], case["D"])
        s["v_pool"] = normal(blocks, case["block"], case["Hkv"], case["D"])
        s["cu_new"] = _cumulative(new)
        s["lens"] = torch.tensor(lens, dtype=torch.int32).cuda()
    else:
        n, v = case["rows"], case["vocab"]
        # a language model's logits: a broad bulk and a few dozen likely tokens
        x = torch.randn((n, v), device="cuda", generator=g) * 2.0
        hot = torch.randint(0, v, (n, 40), device="cuda", generator=g)
        x.scatter_add_(1, hot, torch.rand((n, 40), device="cuda", generator=g) * 10.0)
        s["logits"] = x.to(dtype)

        def pick(values, kind):
            at = torch.randint(0, len(values), (n,), device="cuda", generator=g)
            return torch.tensor(values, dtype=kind).cuda()[at]

        if case["mode"] == "mixed":
            s["temperature"] = pick([0.0, 0.6, 0.8, 1.0, 1.3], torch.float32)
            s["top_k"] = pick([0, 0, 20, 50, 1000], torch.int32)
            s["top_p"] = pick([1.0, 1.0, 0.8, 0.95], torch.float32)
            s["min_p"] = pick([0.0, 0.0, 0.05], torch.float32)
        elif case["mode"] == "filters":
            s["temperature"] = pick([0.7, 1.0], torch.float32)
            s["top_k"] = pick([50, 200], torch.int32)
            s["top_p"] = pick([0.9, 0.95], torch.float32)
            s["min_p"] = pick([0.01, 0.05], torch.float32)
        else:
            s["temperature"] = pick([0.9, 1.1], torch.float32)
            s["top_k"] = torch.zeros(n, dtype=torch.int32, device="cuda")
            s["top_p"] = torch.ones(n, device="cuda")
            s["min_p"] = torch.zeros(n, device="cuda")
        s["u"] = torch.rand(n, device="cuda", generator=g)
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
        if op == "prefill":
            return _B.flash_attn_packed(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
        if op == "decode":
            return _B.flash_attn_paged_batch(s["q"], s["k_pool"], s["v_pool"], s["table"], s["lens"])
        if op == "append":
            _B.paged_kv_append(s["k"], s["v"], s["cu_new"], s["lens"], s["k_pool"], s["v_pool"], s["table"])
            return s["k_pool"], s["v_pool"]
        return _B.sample(s["logits"], s["u"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
    return _PLAIN[op](s)


def _weights(scores, seen):
    """Softmax over the last axis of the entries that `seen` marks; a row with none is zero."""
    scores = torch.where(seen, scores, torch.full_like(scores, -math.inf))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _plain_prefill(s):
    """All packed rows against all packed keys, with a mask of the pairs that may meet."""
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    T, Hq, D = q.shape
    N, Hkv, _ = k.shape
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    i = torch.arange(T, device=q.device)
    j = torch.arange(N, device=q.device)
    si = torch.searchsorted(cu_q, i, right=True) - 1
    sj = torch.searchsorted(cu_k, j, right=True) - 1
    # position of row i among its sequence's keys: the last row sees the last key
    place = i - cu_q[si + 1] + cu_k[si + 1]
    seen = (si[:, None] == sj[None, :]) & (j[None, :] <= place[:, None])
    qh = q.view(T, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
    kh, vh = k.permute(1, 0, 2)[:, None], v.permute(1, 0, 2)[:, None]
    p = _weights(torch.matmul(qh, kh.transpose(-1, -2)) / math.sqrt(D), seen)
    return torch.matmul(p, vh).permute(2, 0, 1, 3).reshape(T, Hq, D).to(s["q"].dtype)


def _plain_decode(s):
    """The pages gathered into one padded batch, then masked attention of one row each."""
    q, table, lens = s["q"].float(), s["table"].long(), s["lens"].long()
    B, Hq, D = q.shape
    block, Hkv = s["k_pool"].shape[1], s["k_pool"].shape[2]
    keys = table.shape[1] * block
    j = torch.arange(keys, device=q.device)
    rows = table[:, j // block] * block + j % block
    kh = s["k_pool"].view(-1, Hkv, D)[rows].float().permute(0, 2, 1, 3)
    vh = s["v_pool"].view(-1, Hkv, D)[rows].float().permute(0, 2, 1, 3)
    qh = q.view(B, Hkv, Hq // Hkv, D)
    seen = (j[None, :] < lens[:, None])[:, None, None, :]
    p = _weights(torch.matmul(qh, kh.transpose(-1, -2)) / math.sqrt(D), seen)
    return torch.matmul(p, vh).reshape(B, Hq, D).to(s["q"].dtype)


def _plain_append(s):
    k_pool, v_pool, cu, lens = s["k_pool"], s["v_pool"], s["cu_new"].long(), s["lens"].long()
    block = k_pool.shape[1]
    t = torch.arange(s["k"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = lens[b] - cu[b + 1] + t
    page = s["table"].long()[b, pos // block]
    k_pool[page, pos % block] = s["k"]
    v_pool[page, pos % block] = s["v"]
    return k_pool, v_pool


def _plain_sample(s):
    """Weights in whole units of 2^-40 of the likeliest token's; every sum is exact.

    Tokens are ordered by logit, equal ones by index. top-k keeps a head of that order,
    top-p the shortest head that holds its share of what top-k kept, min-p what weighs
    at least its share of the likeliest. The draw walks the kept tokens by index.
    """
    x = s["logits"].float()
    n, vocab = x.shape
    cold = (s["temperature"] <= 0)[:, None]
    t = torch.where(cold, torch.ones_like(x[:, :1]), s["temperature"][:, None])
    top = x.amax(-1, keepdim=True)
    weight = torch.floor(torch.exp((x - top) * (1.0 / t)) * 2.0 ** 40).long()
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1]
    w = torch.gather(weight, 1, order)
    rank = torch.arange(vocab, device=x.device)[None]
    k = torch.where(s["top_k"] <= 0, torch.full_like(s["top_k"], vocab), s["top_k"]).long()[:, None]
    k = torch.where(cold, torch.ones_like(k), k)
    w = torch.where(rank < k, w, torch.zeros_like(w))
    run_up = torch.cumsum(w, -1)
    share = (s["top_p"].double()[:, None] * run_up[:, -1:].double()).long()
    everything = s["top_p"][:, None] >= 1
    w = torch.where(everything | (rank == 0) | (run_up - w < share), w, torch.zeros_like(w))
    least = (s["min_p"].double()[:, None] * 2.0 ** 40).long()
    w = torch.where(w >= least, w, torch.zeros_like(w))
    kept = torch.zeros_like(w).scatter_(1, order, w)
    walk = torch.cumsum(kept, -1)
    total = walk[:, -1:]
    at = (s["u"].double()[:, None] * total.double()).long().clamp(min=0)
    at = torch.minimum(at, total - 1)
    return (walk <= at).sum(-1).to(torch.int32)


_PLAIN = {"prefill": _plain_prefill, "decode": _plain_decode, "append": _plain_append, "sample": _plain_sample}


# ---------------------------------------------------------------------------
# what a pass cannot do without

def work(case):
    op, e = case["op"], _BYTES[case["dtype"]]
    if op == "prefill":
        ql, past = _ints(case["q_lens"]), _ints(case["past"])
        keys = sum(ql) + sum(past)
        pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(ql, past))
        return {"bytes": e * case["D"] * (2 * sum(ql) * case["Hq"] + 2 * keys * case["Hkv"]),
                "flops": 4 * case["Hq"] * case["D"] * pairs}
    if op == "decode":
        lens = _ints(case["lens"])
        return {"bytes": e * case["D"] * (2 * sum(lens) * case["Hkv"] + 2 * len(lens) * case["Hq"]),
                "flops": 4 * case["Hq"] * case["D"] * sum(lens)}
    if op == "append":
        return {"bytes": 4 * e * case["D"] * case["Hkv"] * sum(_ints(case["new"])), "flops": 0}
    return {"bytes": e * case["rows"] * case["vocab"], "flops": case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------
# the definition in 64 bits

def _attention64(q, k, v, past):
    """q (n, Hq, D) over k, v (m, Hkv, D): row i sees keys 0 .. past + i."""
    n, Hq, D = q.shape
    m, Hkv, _ = k.shape
    if n == 0 or m == 0:
        return torch.zeros((n, Hq, D), dtype=torch.float64, device=q.device)
    out = torch.empty((n, Hq, D), dtype=torch.float64, device=q.device)
    j = torch.arange(m, device=q.device)
    hidden = j[None, :] > past + torch.arange(n, device=q.device)[:, None]
    for h in range(Hq):
        g = h // (Hq // Hkv)
        a = q[:, h].double() @ k[:, g].double().T / D ** 0.5
        a.masked_fill_(hidden, -math.inf)
        out[:, h] = torch.softmax(a, -1) @ v[:, g].double()
    return out


def exact(case, seed):
    op = case["op"]
    if op == "sample":  # token ids: whole numbers
        return None
    s = prepare(case, seed)
    if op == "prefill":
        cq, ck = s["cu_q"].tolist(), s["cu_k"].tolist()
        past = _ints(case["past"])
        return torch.cat([_attention64(s["q"][cq[b]:cq[b + 1]], s["k"][ck[b]:ck[b + 1]], s["v"][ck[b]:ck[b + 1]],
                                       past[b]) for b in range(len(past))])
    block = case["block"]
    if op == "decode":
        rows = []
        for b, n in enumerate(_ints(case["lens"])):
            pages = s["table"][b, :-(-n // block)].long()
            k = s["k_pool"][pages].flatten(0, 1)[:n]
            v = s["v_pool"][pages].flatten(0, 1)[:n]
            rows.append(_attention64(s["q"][b:b + 1], k, v, n - 1))
        return torch.cat(rows)
    at = 0
    table = s["table"].tolist()
    for b, (n, past) in enumerate(zip(_ints(case["new"]), _ints(case["past"]))):
        done = 0
        while done < n:  # page by page
            pos = past + done
            page, off = table[b][pos // block], pos % block
            step = min(block - off, n - done)
            for pool, rows in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])):
                pool[page, off:off + step] = rows[at + done:at + done + step]
            done += step
        at += n
    return s["k_pool"].double(), s["v_pool"].double()
