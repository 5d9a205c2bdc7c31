"""Measured cases of the ragged-batch operators: attention of one new token over
a paged KV cache, causal attention over packed prompts and over prompt chunks
that continue the cache, the norm + RoPE + page store in front of them, and the
log-probabilities taken from the logits behind them.

``run`` with ``own`` false computes an operator in elementary torch operations
in 32 bits; with ``own`` true it makes the framework's call. ``exact`` is the
operator's definition in 64 bits.
"""

import math
import random

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-6
_THETA = 1_000_000.0


def listed():
    moe = {"nq": 32, "nkv": 4, "dim": 128}    # the head layout of the benchmark model
    mini = {"nq": 16, "nkv": 2, "dim": 64}    # the head layout of the small test model
    return [
        # a single user's first replies: one sequence, a short context, latency only
        {"name": "decode 1 short", "op": "decode", "batch": 1, "lo": 257, "hi": 257, "page": 64,
         "dtype": "bf16", "mix": 1, **moe},
        # one decode step of a mixed batch of 32 conversations, small pages
        {"name": "decode 32 mixed", "op": "decode", "batch": 32, "lo": 128, "hi": 4096, "page": 16,
         "dtype": "bf16", "mix": 2, **moe},
        # documents near the model's position limit: the cache is what is read
        {"name": "decode 16 long", "op": "decode", "batch": 16, "lo": 20000, "hi": 40960,
         "page": 64, "dtype": "bf16", "mix": 3, **moe},
        # one short question
        {"name": "prompt 1 short", "op": "prompt", "prompts": 1, "lo": 37, "hi": 37,
         "dtype": "bf16", "mix": 4, **moe},
        # a batch of 32 prompts as they arrive, from a few words to a page of text
        {"name": "prompt 32 mixed", "op": "prompt", "prompts": 32, "lo": 5, "hi": 1021,
         "dtype": "bf16", "mix": 5, **moe},
        # documents: the attention's own products bound the step
        {"name": "prompt 4 long", "op": "prompt", "prompts": 4, "lo": 1500, "hi": 8192,
         "dtype": "bf16", "mix": 6, **moe},
        # 512-token chunks of 8 prompts that continue what the cache holds
        {"name": "chunk 8", "op": "chunk", "prompts": 8, "lo": 512, "hi": 512, "past_lo": 500,
         "past_hi": 6000, "page": 32, "dtype": "fp16", "mix": 7, **mini},
        # the new tokens of one decode step of 32 sequences
        {"name": "append 32", "op": "append", "tokens": 32, "page": 16, "dtype": "bf16", "mix": 8,
         **moe},
        # the tokens of a prefill of 8000-odd tokens
        {"name": "append 8191", "op": "append", "tokens": 8191, "page": 64, "dtype": "bf16",
         "mix": 9, **moe},
        # the sampled token of one user, with the alternatives an API shows
        {"name": "logprobs 1", "op": "logprobs", "rows": 1, "vocab": 151936, "k": 5,
         "dtype": "bf16", "masked": 0.0},
        # a decode batch; a quarter of the rows under a grammar that allows few tokens
        {"name": "logprobs 33 masked", "op": "logprobs", "rows": 33, "vocab": 151936, "k": 20,
         "dtype": "fp32", "masked": 0.25},
        # scoring of prompts
        {"name": "logprobs 4096", "op": "logprobs", "rows": 4096, "vocab": 151936, "k": 8,
         "dtype": "bf16", "masked": 0.0},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["decode", "prompt", "chunk", "append", "logprobs"])
    dim = rng.choice([64, 128])
    nkv = rng.choice([1, 2, 4, 8])
    heads = {"nkv": nkv, "nq": nkv * rng.choice([1, 2, 3, 4, 5, 7, 8]), "dim": dim}
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    mix = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if op == "decode":
        hi = _log_int(rng, 1, 40960)
        # no more cache bytes than the largest listed case can hold
        most = max(1, min(256, (16 * 40960 * 4 * 128) // (2 * hi * nkv * dim)))
        return {"op": op, "batch": _log_int(rng, 1, most), "lo": rng.choice([0, max(1, hi // 8)]),
                "hi": hi, "page": page, "dtype": dtype, "mix": mix, **heads}
    if op == "prompt":
        hi = _log_int(rng, 1, 6000)
        return {"op": op, "prompts": _log_int(rng, 1, max(1, min(64, 12000 // hi))),
                "lo": max(1, hi // rng.choice([1, 4, 100])), "hi": hi, "dtype": dtype, "mix": mix,
                **{**heads, "nq": min(heads["nq"], 4 * nkv if nkv == 8 else heads["nq"])}}
    if op == "chunk":
        hi = _log_int(rng, 1, 1024)
        return {"op": op, "prompts": _log_int(rng, 1, 8), "lo": max(1, hi // 3), "hi": hi,
                "past_lo": 0, "past_hi": _log_int(rng, 1, 6000), "page": page, "dtype": dtype,
                "mix": mix, **{**heads, "nq": min(heads["nq"], 32)}}
    if op == "append":
        return {"op": op, "tokens": _log_int(rng, 1, 8191), "page": page, "dtype": dtype,
                "mix": mix, **{**heads, "nq": min(heads["nq"], 32)}}
    vocab = _log_int(rng, 1000, 151936)
    return {"op": op, "rows": _log_int(rng, 1, min(4096, 4096 * 75000 // vocab)), "vocab": vocab,
            "k": rng.choice([0, 1, 5, 20]), "dtype": rng.choice(["bf16", "fp16", "fp32"]),
            "masked": rng.choice([0.0, 0.5])}


# ------------------------------------------------------------------- sizes --
def _lengths(n, lo, hi, mix):
    """n lengths spread over the logarithm of [lo, hi]; the longest is hi."""
    r = random.Random(mix)
    got = [min(hi, max(lo, int(math.exp(r.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))
           for _ in range(n)]
    if lo == 0:
        got = [0 if r.random() < 0.1 else g for g in got]
    got[r.randrange(n)] = hi
    return got


def _past(case):
    r = random.Random(case["mix"] + 1)
    return [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["prompts"])]


def work(case):
    op, e = case["op"], _SIZE[case["dtype"]]
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * e + case["rows"] * (16 + 12 * case["k"]), "flops": 4 * n}
    nq, nkv, d = case["nq"], case["nkv"], case["dim"]
    if op == "append":
        t = case["tokens"]
        # qkv in, q out, k and v into their pages, one table row a token
        return {"bytes": t * ((nq + 2 * nkv) * d * e * 2 + 4 * d + 12),
                "flops": t * (nq + nkv) * d * 8}
    if op == "decode":
        ln = _lengths(case["batch"], case["lo"], case["hi"], case["mix"])
        kv = sum(ln)
        return {"bytes": kv * nkv * d * e * 2 + case["batch"] * nq * d * e * 2,
                "flops": 4 * kv * nq * d}
    ln = _lengths(case["prompts"], case["lo"], case["hi"], case["mix"])
    past = _past(case) if op == "chunk" else [0] * len(ln)
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(ln, past))
    rows, keys = sum(ln), sum(ln) + sum(past)
    return {"bytes": (2 * rows * nq + 2 * keys * nkv) * d * e, "flops": 4 * pairs * nq * d}


# ------------------------------------------------------------------ inputs --
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(_DT[dtype])


def _pool(g, case, lens):
    """Pages that hold `lens` tokens in a scattered order, and the page table."""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32).cpu()
    table = torch.zeros(len(lens), max(max(need), 1), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    shape = (total, case["nkv"], page, case["dim"])
    return {"k_pages": _randn(g, shape, case["dtype"]), "v_pages": _randn(g, shape, case["dtype"]),
            "page_table": table.to(DEV),
            "seq_lens": torch.tensor(lens, dtype=torch.int32, device=DEV)}


def prepare(case, seed):
    op, g = case["op"], _gen(seed)
    s = {"case": dict(case)}
    if op == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.empty(rows, vocab, device=DEV, dtype=_DT[case["dtype"]])
        for a in range(0, rows, 512):  # logits of a few units' spread with some likely tokens
            b = min(rows, a + 512)
            part = torch.randn(b - a, vocab, generator=g, device=DEV) * 2.5
            hot = torch.randint(vocab, (b - a, 8), generator=g, device=DEV)
            part.scatter_add_(1, hot, torch.rand(b - a, 8, generator=g, device=DEV) * 14)
            if case["masked"]:  # rows in which a mask leaves 30 tokens
                keep = torch.zeros(b - a, vocab, dtype=torch.bool, device=DEV)
                keep.scatter_(1, torch.randint(vocab, (b - a, 30), generator=g, device=DEV), True)
                keep |= (torch.rand(b - a, 1, generator=g, device=DEV) >= case["masked"])
                part.masked_fill_(~keep, float("-inf"))
            x[a:b] = part.to(x.dtype)
        s["logits"] = x
        some = torch.randint(vocab, (rows,), generator=g, device=DEV)
        best = x.argmax(-1)
        # mostly the likely token, sometimes any token that the mask allows
        pick = (torch.rand(rows, generator=g, device=DEV) < 0.3) & torch.isfinite(
            x.gather(1, some[:, None])[:, 0])
        s["ids"] = torch.where(pick, some, best)
        return s
    nq, nkv, d, dt = case["nq"], case["nkv"], case["dim"], case["dtype"]
    if op == "append":
        t, page = case["tokens"], case["page"]
        s["qkv"] = _randn(g, (t, (nq + 2 * nkv) * d), dt, 1.5)
        s["q_norm"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(_DT[dt])
        s["k_norm"] = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(_DT[dt])
        span = 8192
        ang = torch.arange(span, device=DEV, dtype=torch.float32)[:, None] * (
            1.0 / _THETA ** (torch.arange(0, d, 2, device=DEV).float() / d))[None, :]
        s["rope"] = torch.cat([ang.cos(), ang.sin()], -1).contiguous()
        first = random.Random(case["mix"]).randint(0, span - t)
        s["positions"] = torch.arange(first, first + t, device=DEV, dtype=torch.int32)
        pages = -(-t // page) + 2
        order = torch.randperm(pages, generator=g, device=DEV)
        at = torch.arange(t, device=DEV)
        s["slots"] = order[at // page] * page + at % page
        shape = (pages, nkv, page, d)
        s["k_pages"], s["v_pages"] = _randn(g, shape, dt), _randn(g, shape, dt)
        return s
    if op == "decode":
        lens = _lengths(case["batch"], case["lo"], case["hi"], case["mix"])
        s.update(_pool(g, case, lens))
        s["q"] = _randn(g, (case["batch"], nq, d), dt, 1.5)
        return s
    lens = _lengths(case["prompts"], case["lo"], case["hi"], case["mix"])
    rows = sum(lens)
    s["lens"] = lens
    s["q"] = _randn(g, (rows, nq, d), dt, 1.5)
    s["cu_seqlens"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    if op == "chunk":
        s["past"] = _past(case)
        s.update(_pool(g, case, [n + p for n, p in zip(lens, s["past"])]))
    else:
        s["k"] = _randn(g, (rows, nkv, d), dt)
        s["v"] = _randn(g, (rows, nkv, d), dt)
    return s


# --------------------------------------------------------------- plain forms --
def _soft(sc, seen):
    """Weights of the scores `sc` (overwritten) over the keys in `seen`; none
    for a row that sees no key."""
    sc.masked_fill_(~seen, float("-inf"))
    m = sc.amax(-1, keepdim=True)
    sc.sub_(torch.where(torch.isfinite(m), m, torch.zeros_like(m))).exp_()
    return sc.div_(sc.sum(-1, keepdim=True).clamp_min(1e-30))


def _plain_decode(s):
    c = s["case"]
    b, nkv, d = c["batch"], c["nkv"], c["dim"]
    table = s["page_table"].long()
    k = s["k_pages"][table].permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, d).float()
    v = s["v_pages"][table].permute(0, 2, 1, 3, 4).reshape(b, nkv, -1, d).float()
    q = s["q"].view(b, nkv, -1, d).float()
    sc = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(d)
    seen = torch.arange(k.shape[2], device=DEV)[None, :] < s["seq_lens"][:, None]
    p = _soft(sc, seen[:, None, None, :])
    return torch.matmul(p, v).to(s["q"].dtype).reshape(b, -1)


def _plain_rows(q, k, v):
    """q [n, nq, d] at the last n of the m positions of k, v [nkv, m, d]."""
    n, nq, d = q.shape
    nkv, m, _ = k.shape
    qf = q.float().view(n, nkv, nq // nkv, d).permute(1, 2, 0, 3).reshape(nkv, -1, d)
    sc = torch.matmul(qf, k.transpose(-1, -2)).div_(math.sqrt(d)).view(nkv, -1, n, m)
    at = torch.arange(m, device=DEV)
    p = _soft(sc, at[None, :] <= at[m - n:, None]).view(nkv, -1, m)
    return torch.matmul(p, v).view(nkv, -1, n, d).permute(2, 0, 1, 3).reshape(n, nq * d).to(q.dtype)


def _plain_prompt(s):
    got, a = [], 0
    for i, n in enumerate(s["lens"]):
        q = s["q"][a:a + n]
        if "past" in s:
            c, m = s["case"], n + s["past"][i]
            t = s["page_table"][i, : -(-m // c["page"])].long()
            k, v = (s[x][t].transpose(0, 1).reshape(c["nkv"], -1, c["dim"])[:, :m].float()
                    for x in ("k_pages", "v_pages"))
        else:
            k, v = (s[x][a:a + n].transpose(0, 1).float() for x in ("k", "v"))
        got.append(_plain_rows(q, k, v))
        a += n
    return torch.cat(got)


def _plain_append(s):
    c = s["case"]
    nq, nkv, d = c["nq"], c["nkv"], c["dim"]
    x = s["qkv"].view(-1, nq + 2 * nkv, d)
    qk = x[:, : nq + nkv].float()
    w = torch.cat([s["q_norm"].expand(nq, d), s["k_norm"].expand(nkv, d)]).float()
    qk = qk * torch.rsqrt(qk.pow(2).mean(-1, keepdim=True) + _EPS) * w
    cs = s["rope"][s["positions"].long()][:, None, :]
    cos, sin = cs[..., : d // 2], cs[..., d // 2:]
    lo, hi = qk[..., : d // 2], qk[..., d // 2:]
    qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).to(s["qkv"].dtype)
    page, off = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_pages"][page, :, off] = qk[:, nq:]
    s["v_pages"][page, :, off] = x[:, nq + nkv:]
    return qk[:, :nq].reshape(-1, nq * d), s["k_pages"], s["v_pages"]


def _plain_logprobs(s):
    k = s["case"]["k"]
    x = s["logits"].float()
    m = x.amax(-1, keepdim=True)
    sh = x - m
    e = sh.exp()
    z = e.sum(-1, keepdim=True)
    lse = m + z.log()
    ent = z.log() - (e * sh.clamp_min(-1e30)).sum(-1, keepdim=True) / z
    got = [(x.gather(1, s["ids"][:, None]) - lse)[:, 0], ent[:, 0]]
    if k:
        del sh, e
        # the larger logit first, the lower index first among equal ones
        bits = (x + 0.0).view(torch.int32).long()
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = (bits << 32) - torch.arange(x.shape[1], device=DEV)
        top = key.topk(k, dim=-1).indices
        got += [top, x.gather(1, top) - lse]
    return tuple(got)


def run(state):
    c = state["case"]
    op = c["op"]
    if own:
        from afd_demo_b200 import ops
        if op == "decode":
            return ops.paged_decode_attention(state["q"], state["k_pages"], state["v_pages"],
                                              state["page_table"], state["seq_lens"])
        if op == "prompt":
            return ops.packed_attention(state["q"], state["k"], state["v"], state["cu_seqlens"])
        if op == "chunk":
            return ops.paged_prefill_attention(state["q"], state["k_pages"], state["v_pages"],
                                               state["page_table"], state["seq_lens"],
                                               state["cu_seqlens"])
        if op == "append":
            q = ops.qk_norm_rope_paged(state["qkv"], state["q_norm"], state["k_norm"],
                                       state["rope"], state["k_pages"], state["v_pages"],
                                       state["positions"], state["slots"], c["nq"], c["nkv"],
                                       _EPS)
            return q.view(c["tokens"], -1), state["k_pages"], state["v_pages"]
        r = ops.token_logprobs(state["logits"], state["ids"], top_k=c["k"])
        return ((r.logprob, r.entropy, r.top_ids, r.top_logprobs) if c["k"]
                else (r.logprob, r.entropy))
    return {"decode": _plain_decode, "prompt": _plain_prompt, "chunk": _plain_prompt,
            "append": _plain_append, "logprobs": _plain_logprobs}[op](state)


# ------------------------------------------------------------------- 64 bits --
def _exact_row_block(q, k, v, seen):
    """softmax(q k^T / sqrt d) v for one query head, rows of `q` over the keys of
    `k`; seen[r] = how many of the first keys row r sees."""
    sc = q @ k.T * (q.shape[-1] ** -0.5)
    at = torch.arange(k.shape[0], device=DEV)
    sc = torch.where(at[None, :] < seen[:, None], sc, torch.full_like(sc, -torch.inf))
    return torch.nan_to_num(torch.softmax(sc, -1)) @ v


def _exact_attention(case, s):
    op, nq, nkv, d = case["op"], case["nq"], case["nkv"], case["dim"]
    q = s["q"].double()
    out = torch.zeros_like(q)
    news = [1] * case["batch"] if op == "decode" else s["lens"]
    row = 0
    for i, n in enumerate(news):
        if op == "prompt":
            keys, vals, m = s["k"][row:row + n], s["v"][row:row + n], n
        else:
            m = int(s["seq_lens"][i])
            pos = torch.arange(m, device=DEV)
            page = s["page_table"][i].long()[pos // case["page"]]
            keys = s["k_pages"][page, :, pos % case["page"]]
            vals = s["v_pages"][page, :, pos % case["page"]]
        if m:
            seen = torch.arange(m - n + 1, m + 1, device=DEV)
            for h in range(nq):
                kh = h // (nq // nkv)
                out[row:row + n, h] = _exact_row_block(q[row:row + n, h], keys[:, kh].double(),
                                                       vals[:, kh].double(), seen)
        row += n
    return out.reshape(q.shape[0], nq * d)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("decode", "prompt", "chunk"):
        return _exact_attention(case, s)
    if op == "append":
        nq, nkv, d, page = case["nq"], case["nkv"], case["dim"], case["page"]
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        x = s["qkv"].double().reshape(-1, nq + 2 * nkv, d)
        turn = s["rope"].double()[s["positions"].long()]
        z = torch.complex(turn[:, : d // 2], turn[:, d // 2:])[:, None]  # cos + i sin

        def normed(heads, weight):
            y = heads / (heads.square().sum(-1, keepdim=True) / d + _EPS).sqrt() * weight.double()
            y = torch.complex(y[..., : d // 2].contiguous(), y[..., d // 2:].contiguous()) * z
            return torch.cat([y.real, y.imag], -1)

        where = (s["slots"] // page, slice(None), s["slots"] % page)
        kp[where] = normed(x[:, nq:nq + nkv], s["k_norm"])
        vp[where] = x[:, nq + nkv:]
        return normed(x[:, :nq], s["q_norm"]).reshape(-1, nq * d), kp, vp
    lp, ent, top = [], [], []
    for a in range(0, case["rows"], 256):
        x = s["logits"][a:a + 256].double()
        ls = x - torch.logsumexp(x, -1, keepdim=True)
        lp.append(ls[torch.arange(ls.shape[0], device=DEV), s["ids"][a:a + 256]])
        ent.append(torch.special.entr(ls.exp()).sum(-1))
        top.append(ls.topk(case["k"], -1).values)
    got = (torch.cat(lp), torch.cat(ent))
    return got + (None, torch.cat(top)) if case["k"] else got
