"""What is timed and compared of the ragged-batch operators: planning a step over requests with any number
of new tokens each (``ragged_plan``), norms + rotary positions + paged K/V append (``norm_rope_kv_append``),
causal attention of the packed new tokens over the paged cache (``ragged_attn``), and verification of drafted
tokens against the target's probabilities (``verify_drafts``).

``run`` computes an operator in plain torch operations while ``own`` is False and calls the package's
operator while it is True; ``exact`` restates the definition in 64 bits. Sizes are this repository's model
shapes (24/8 heads of 128, 14/2 and 12/12 heads of 64; vocabularies of 128256, 151936 and 50257) or generic.
"""

import math
import random

import numpy as np
import torch

own = False

BLOCK = 16


# ---- cases -------------------------------------------------------------------------------------------

def listed():
    return [
        # attention: one request decoding its next token over a long cache (latency, split over the cache)
        dict(name="attn_one_token", op="attn", b=1, q_lo=1, q_hi=1, ctx_lo=32763, ctx_hi=32763, hq=24, hkv=8, d=128,
             kv8=False, shape=1),
        # attention: a serving step that verifies four drafted tokens of every running request
        dict(name="attn_verify", op="attn", b=32, q_lo=5, q_hi=5, ctx_lo=300, ctx_hi=4000, hq=24, hkv=8, d=128,
             kv8=False, shape=2),
        # attention: prompts of different lengths packed into one pass, heads of 64 with a group of seven
        dict(name="attn_packed_prompts", op="attn", b=24, q_lo=17, q_hi=2047, ctx_lo=0, ctx_hi=0, hq=14, hkv=2, d=64,
             kv8=False, shape=3),
        # attention: a continuous-batching step on an INT8 cache, prompt chunks beside single tokens
        dict(name="attn_chunks_kv8", op="attn", b=16, q_lo=1, q_hi=700, ctx_lo=10, ctx_hi=6000, hq=24, hkv=8, d=128,
             kv8=True, shape=4),
        # attention: one long prompt
        dict(name="attn_long_prompt", op="attn", b=1, q_lo=8192, q_hi=8192, ctx_lo=0, ctx_hi=0, hq=24, hkv=8, d=128,
             kv8=False, shape=5),
        # plan: a decoding step with a few drafted tokens each
        dict(name="plan_step", op="plan", b=32, q_lo=1, q_hi=8, ctx_lo=1, ctx_hi=4000, pad=7, shape=6),
        # plan: the largest, many requests with prompts of every length
        dict(name="plan_prompts", op="plan", b=1000, q_lo=1, q_hi=333, ctx_lo=0, ctx_hi=900, pad=100, shape=7),
        # append: the verify step's rows, query and key norms
        dict(name="append_step", op="append", rows=160, hq=24, hkv=8, d=128, norm=True, rope=True, kv8=False),
        # append: the packed prompts' rows onto an INT8 cache, norms
        dict(name="append_prompts_kv8", op="append", rows=5003, hq=14, hkv=2, d=64, norm=True, rope=True, kv8=True),
        # append: the long prompt's rows, rotation only
        dict(name="append_long_prompt", op="append", rows=8192, hq=24, hkv=8, d=128, norm=False, rope=True, kv8=False),
        # verify: one request, drafts without probabilities (copied from its prompt)
        dict(name="verify_one", op="verify", b=1, k_lo=4, k_hi=4, vocab=50257, probs=False, shape=11),
        # verify: a full batch with a draft model's probabilities, greedy and sampled requests mixed
        dict(name="verify_batch", op="verify", b=48, k_lo=1, k_hi=8, vocab=128256, probs=True, shape=12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["attn", "attn", "attn", "plan", "append", "append", "verify", "verify"])
    shape = rng.randrange(1 << 30)
    heads = [(24, 8, 128), (14, 2, 64), (12, 12, 64), (32, 4, 128), (16, 1, 64), (6, 6, 32), (3, 1, 128)]
    if op == "attn":
        hq, hkv, d = rng.choice(heads)
        while True:
            b = _log(rng, 1, 48)
            q_hi = _log(rng, 1, 8192)
            ctx_hi = rng.choice([0, _log(rng, 1, 32768)])
            c = dict(op="attn", b=b, q_lo=rng.choice([1, max(1, q_hi // 3), q_hi]), q_hi=q_hi,
                     ctx_lo=rng.choice([0, ctx_hi]), ctx_hi=ctx_hi, hq=hq, hkv=hkv, d=d, kv8=rng.random() < 0.35,
                     shape=shape)
            w, top = work(c), work(listed()[4])
            n, t = (max(x) for x in _lens(c))
            padded = 4 * b * (n + t + BLOCK) * max(hq * n, 2 * hkv * d)  # the plain form's largest arrays
            if w["flops"] <= top["flops"] and w["bytes"] <= 3e8 and padded <= 8e9:
                return c
    if op == "plan":
        b = _log(rng, 1, 1000)
        q_hi = _log(rng, 1, max(2, 160000 // b if b > 400 else 333))
        return dict(op="plan", b=b, q_lo=1, q_hi=min(q_hi, 333), ctx_lo=0, ctx_hi=_log(rng, 1, 4000 if b < 400 else 900),
                    pad=rng.choice([0, rng.randrange(1, 100)]), shape=shape)
    if op == "append":
        hq, hkv, d = rng.choice(heads)
        most = 8192 * 40 * 128 // ((hq + 2 * hkv) * d)
        return dict(op="append", rows=_log(rng, 1, min(most, 8192)), hq=hq, hkv=hkv, d=d, norm=rng.random() < 0.6,
                    rope=rng.random() < 0.8, kv8=rng.random() < 0.4)
    vocab = rng.choice([50257, 128256, 151936, _log(rng, 500, 40000)])
    return dict(op="verify", b=_log(rng, 1, 40), k_lo=rng.choice([0, 1]), k_hi=rng.randrange(1, 9), vocab=vocab,
                probs=rng.random() < 0.6, shape=shape)


def _lens(case):
    """New tokens and cached tokens of every request, spread over the logarithm of the case's ranges."""
    rng = random.Random(case["shape"])
    q, ctx = [], []
    for _ in range(case["b"]):
        q.append(_log(rng, case["q_lo"], case["q_hi"]))
        ctx.append(_log(rng, case["ctx_lo"] + 1, case["ctx_hi"] + 1) - 1)
    return q, ctx


def _drafts(case):
    rng = random.Random(case["shape"])
    return [rng.randint(case["k_lo"], case["k_hi"]) for _ in range(case["b"])]


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _starts(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


# ---- inputs ------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    return {"attn": _prepare_attn, "plan": _prepare_plan, "append": _prepare_append,
            "verify": _prepare_verify}[case["op"]](case, g, rng)


def _i32(a):
    return torch.as_tensor(np.asarray(a, dtype=np.int32), device="cuda")


def _codes(g, n, hkv, d):
    """An INT8 cache as the append kernel leaves it: codes of unit-variance vectors and their scales."""
    x = torch.randn((n, hkv, BLOCK, d), generator=g, device="cuda")
    s = x.abs().amax(-1) / 127.0
    return torch.round(x / s[..., None]).clamp_(-128, 127).to(torch.int8), s


def _prepare_attn(case, g, rng):
    q_lens, ctx = _lens(case)
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    need = [_blocks(c + n) for c, n in zip(ctx, q_lens)]
    n_blocks = sum(need) + 5
    perm = rng.permutation(n_blocks).astype(np.int32)
    tables = np.zeros((b, max(need)), np.int32)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = perm[at:at + n]
        at += n
    st = dict(case=case, q_lens=q_lens, ctx=ctx, scale=1.0 / math.sqrt(d), tables=_i32(tables))
    row = np.concatenate([i * max(q_lens) + np.arange(n) for i, n in enumerate(q_lens)])
    st["at"] = torch.as_tensor(row, device="cuda")
    st["first"] = torch.as_tensor(ctx, device="cuda")
    st["kv"] = torch.as_tensor([c + n for c, n in zip(ctx, q_lens)], device="cuda")
    st["q"] = torch.randn((sum(q_lens), hq, d), generator=g, device="cuda").to(torch.bfloat16)
    if case["kv8"]:
        st["k"], st["ks"] = _codes(g, n_blocks, hkv, d)
        st["v"], st["vs"] = _codes(g, n_blocks, hkv, d)
    else:
        st["k"] = torch.randn((n_blocks, hkv, BLOCK, d), generator=g, device="cuda").to(torch.bfloat16)
        st["v"] = torch.randn((n_blocks, hkv, BLOCK, d), generator=g, device="cuda").to(torch.bfloat16)
    if own:  # the step's plan, which serves the attention of every layer
        from microgen_b200 import kernels as K
        st["plan"] = K.RaggedPlan(b, sum(q_lens), tables.shape[1], hq, hkv, d, "cuda")
        K.ragged_plan(st["plan"], _i32(q_lens), _i32(ctx), st["tables"], n_blocks)
    return st


def _prepare_plan(case, g, rng):
    q_lens, ctx = _lens(case)
    b = case["b"]
    have = [_blocks(c) for c in ctx]
    need = [_blocks(c + n) for c, n in zip(ctx, q_lens)]
    for i in range(b):  # a rolled-back request still holds the blocks of its rejected tokens
        if rng.random() < 0.2:
            have[i] = min(need[i], have[i] + 1)
    width = max(need) + 3
    fresh = sum(n - h for n, h in zip(need, have))
    total = sum(have) + fresh + 40
    perm = rng.permutation(total).astype(np.int32)
    tables = np.zeros((b, width), np.int32)
    at = 0
    for i, n in enumerate(have):
        tables[i, :n] = perm[at:at + n]
        at += n
    cursor = int(rng.integers(0, 30))
    free = np.concatenate([np.zeros(cursor, np.int32), perm[at:]])
    st = dict(case=case, rows=sum(q_lens) + case["pad"], num_blocks=total, q_lens=_i32(q_lens), ctx=_i32(ctx),
              tables=_i32(tables), n_blocks=_i32(have), free=_i32(free), cursor=_i32([cursor]))
    if own:
        from microgen_b200 import kernels as K
        st["plan"] = K.RaggedPlan(b, st["rows"], width, 24, 8, 128, "cuda")
    return st


def _rope_table(d, n):
    inv = 1.0 / (500000.0 ** (torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d))
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv[None]
    return torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()


def _prepare_append(case, g, rng):
    r, hq, hkv, d = case["rows"], case["hq"], case["hkv"], case["d"]
    n_blocks = _blocks(r) + 9
    slots = rng.permutation(n_blocks)[:_blocks(r)].repeat(BLOCK)[:r] * BLOCK + np.arange(r) % BLOCK
    start = int(rng.integers(0, 4000))
    st = dict(case=case, slots=_i32(slots), positions=_i32(start + np.arange(r)), eps=1e-6)
    st["qkv"] = torch.randn((r, (hq + 2 * hkv) * d), generator=g, device="cuda") * 1.7
    st["cos_sin"] = _rope_table(d, start + r + 1) if case["rope"] else None
    st["qw"] = st["kw"] = None
    if case["norm"]:
        st["qw"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
        st["kw"] = 1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")
    dt = torch.int8 if case["kv8"] else torch.bfloat16
    st["k"] = torch.zeros((n_blocks, hkv, BLOCK, d), dtype=dt, device="cuda")
    st["v"] = torch.zeros((n_blocks, hkv, BLOCK, d), dtype=dt, device="cuda")
    if case["kv8"]:
        st["ks"] = torch.zeros((n_blocks, hkv, BLOCK), device="cuda")
        st["vs"] = torch.zeros((n_blocks, hkv, BLOCK), device="cuda")
    return st


def _prepare_verify(case, g, rng):
    k = _drafts(case)
    b, vocab = case["b"], case["vocab"]
    rows = sum(k) + b
    cu = _starts([n + 1 for n in k])
    base = torch.randn((rows, vocab), generator=g, device="cuda")
    logits = base * 2.5
    draft = torch.softmax(logits + 0.7 * torch.randn((rows, vocab), generator=g, device="cuda"), -1)
    drawn = torch.multinomial(draft, 1, generator=g)[:, 0]
    temps = np.full(b, 0.8, np.float32)
    temps[1::3] = 1.0
    temps[2::5] = 0.0  # greedy
    best = logits.argmax(-1)
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    greedy = np.repeat(temps == 0.0, np.asarray(k) + 1)
    pick = torch.where(torch.as_tensor(greedy, device="cuda"), best, drawn)
    last = np.zeros(rows, bool)
    last[np.asarray(cu[1:]) - 1] = True
    src = np.nonzero(~last)[0]  # draft j of a request is fed at the row after the one that predicts it
    if len(src):
        tokens[torch.as_tensor(src + 1, device="cuda")] = pick[torch.as_tensor(src, device="cuda")]
    return dict(case=case, k=k, cu=_i32(cu), logits=logits, tokens=tokens.to(torch.int32),
                probs=draft if case["probs"] else None,
                uniforms=torch.rand(rows, generator=g, device="cuda"),
                temps=torch.as_tensor(temps, device="cuda"))


# ---- one pass ----------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"attn": _own_attn, "plan": _own_plan, "append": _own_append, "verify": _own_verify}[op](state)
    return {"attn": _plain_attn, "plan": _plain_plan, "append": _plain_append, "verify": _plain_verify}[op](state)


def _own_attn(s):
    from microgen_b200 import kernels as K
    return K.ragged_attn(s["q"], s["k"], s["v"], s["plan"], s["scale"], k_scales=s.get("ks"), v_scales=s.get("vs"))


def _own_plan(s):
    from microgen_b200 import kernels as K
    p = K.ragged_plan(s["plan"], s["q_lens"], s["ctx"], s["tables"], s["num_blocks"], n_blocks=s["n_blocks"],
                      free_blocks=s["free"], cursor=s["cursor"])
    return [p.cu_rows, p.kv_lens, p.positions, p.slots, p.seq_ids, s["tables"], p.n_blocks, p.cursor]


def _own_append(s):
    from microgen_b200 import kernels as K
    c = s["case"]
    q = K.norm_rope_kv_append(s["qkv"], s["positions"], s["cos_sin"], s["slots"], c["hq"], c["hkv"], c["d"], s["k"],
                              s["v"], q_weight=s["qw"], k_weight=s["kw"], eps=s["eps"], k_scales=s.get("ks"),
                              v_scales=s.get("vs"))
    return _append_out(s, q)


def _append_out(s, q):
    if not s["case"]["kv8"]:
        return [q, s["k"], s["v"]]
    # 8-bit codes as the values they stand for, in the type of an unquantized cache
    k, v = (torch.mul(s[n], s[n + "s"][..., None], out=torch.empty_like(s[n], dtype=torch.bfloat16)) for n in ("k", "v"))
    return [q, k, v, s["ks"], s["vs"]]


def _own_verify(s):
    from microgen_b200 import kernels as K
    return K.verify_drafts(s["logits"], s["tokens"], s["cu"], s["uniforms"], draft_probs=s["probs"],
                           temperatures=s["temps"])


# ---- plain forms -------------------------------------------------------------------------------------

def _cache(s, name):
    """fp32 [b, hkv, tokens, d]: every request's cached tokens, padded to the widest block table."""
    ids = s["tables"].long()
    x = s[name][ids].float()
    if s["case"]["kv8"]:
        x = x * s[name + "s"][ids][..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _plain_attn(s):
    c = s["case"]
    b, hq, hkv, d = c["b"], c["hq"], c["hkv"], c["d"]
    kk, vv = _cache(s, "k"), _cache(s, "v")
    n = max(s["q_lens"])
    q = torch.zeros((b * n, hq, d), device="cuda")
    q[s["at"]] = s["q"].float()  # request i's new tokens are rows i*n and on
    q = q.view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    sc = torch.matmul(q, kk.transpose(2, 3)).view(b, hkv, hq // hkv, n, -1).mul_(s["scale"])
    key = torch.arange(kk.shape[2], device="cuda")
    pos = s["first"][:, None] + torch.arange(n, device="cuda")[None]
    hidden = (key[None, None] > pos[..., None]) | (key[None, None] >= s["kv"][:, None, None])
    sc.masked_fill_(hidden[:, None, None], -math.inf)
    p = sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    vv = torch.where((key[None] < s["kv"][:, None])[:, None, :, None], vv, 0.0)
    o = torch.matmul(p.flatten(2, 3), vv).view(b, hkv, hq // hkv, n, d) / p.sum(-1, keepdim=True)
    return o.permute(0, 3, 1, 2, 4).reshape(b * n, hq * d)[s["at"]].to(torch.bfloat16)


def _plain_plan(s):
    q, ctx, have = s["q_lens"].long(), s["ctx"].long(), s["n_blocks"].long()
    b, rows = q.shape[0], s["rows"]
    cu = torch.cat([q.new_zeros(1), q.cumsum(0)])
    kv = ctx + q
    need = torch.maximum(have, (kv + BLOCK - 1) // BLOCK)
    fresh = need - have
    first = fresh.cumsum(0) - fresh + s["cursor"].long()
    cols = torch.arange(s["tables"].shape[1], device="cuda")[None]
    new = (cols >= have[:, None]) & (cols < need[:, None])
    idx = (first[:, None] + cols - have[:, None]).clamp(0, s["free"].shape[0] - 1)
    s["tables"].copy_(torch.where(new, s["free"][idx], s["tables"]))
    r = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    live = seq < b
    sq = seq.clamp(max=b - 1)
    pos = torch.where(live, ctx[sq] + r - cu[sq], 0)
    slot = s["tables"][sq, pos // BLOCK].long() * BLOCK + pos % BLOCK
    i32 = torch.int32
    return [cu.to(i32), kv.to(i32), pos.to(i32), torch.where(live, slot, -1).to(i32), torch.where(live, seq, -1).to(i32),
            s["tables"], need.to(i32), (s["cursor"] + fresh.sum()).to(i32)]


def _plain_append(s):
    c = s["case"]
    r, hq, hkv, d = c["rows"], c["hq"], c["hkv"], c["d"]
    x = s["qkv"].float().view(r, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + s["eps"]) * s["qw"]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + s["eps"]) * s["kw"]
    if c["rope"]:
        cs = s["cos_sin"][s["positions"].long()][:, None]
        co, si = cs[..., :d // 2], cs[..., d // 2:]

        def turn(t):
            a, e = t[..., :d // 2], t[..., d // 2:]
            return torch.cat([a * co - e * si, e * co + a * si], -1)
        q, k = turn(q), turn(k)
    blk, off = s["slots"].long() // BLOCK, s["slots"].long() % BLOCK
    for name, t in (("k", k), ("v", v)):
        if c["kv8"]:
            sc = (t.abs().amax(-1) / 127.0).clamp(min=1e-8)
            s[name][blk, :, off] = torch.round(t / sc[..., None]).clamp(-128, 127).to(torch.int8)
            s[name + "s"][blk, :, off] = sc
        else:
            s[name][blk, :, off] = t.to(torch.bfloat16)
    return _append_out(s, q.to(torch.bfloat16))


def _plain_verify(s):
    # 64 bits: the sampled index is where a cumulative sum over the vocabulary passes a uniform number
    b = s["cu"].shape[0] - 1
    cu = s["cu"].long()
    n = cu[1:] - cu[:-1] - 1
    rows, vocab = s["logits"].shape
    owner = torch.repeat_interleave(torch.arange(b, device="cuda"), n + 1, output_size=rows)
    t = s["temps"].double()[owner]
    greedy = t == 0
    z = s["logits"].double() / torch.where(greedy, 1.0, t)[:, None]
    p = torch.exp(z - z.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    best = s["logits"].argmax(-1)
    nxt = torch.cat([s["tokens"][1:], s["tokens"][:1]]).long()  # the draft each row is asked about
    pd = p.gather(1, nxt[:, None])[:, 0]
    qd = torch.ones_like(pd) if s["probs"] is None else s["probs"].gather(1, nxt[:, None])[:, 0].double()
    ok = torch.where(greedy, nxt == best, s["uniforms"].double() * qd < pd)
    ok &= torch.arange(rows, device="cuda") != cu[1:][owner] - 1
    r = torch.arange(rows, device="cuda")
    stop = torch.where(ok, rows, r)
    stop = torch.full((b,), rows, device="cuda").scatter_reduce(0, owner, stop, "amin")
    acc = stop - cu[:-1]
    w = p[stop]
    cut = acc < n
    if s["probs"] is None:
        gone = torch.zeros_like(w).scatter_(1, nxt[stop][:, None], 1.0)
    else:
        gone = s["probs"][stop].double()
    rest = torch.where(cut[:, None], (w - gone).clamp(min=0), w)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    c = rest.cumsum(-1)
    hit = c > s["uniforms"].double()[cu[1:] - 1][:, None] * c[:, -1:]
    hit &= rest > 0
    tok = hit.to(torch.uint8).argmax(-1)
    last = vocab - 1 - (rest > 0).flip(-1).to(torch.uint8).argmax(-1)
    tok = torch.where(hit.any(-1), tok, last)
    tok = torch.where(greedy[stop], best[stop], tok)
    return [acc.to(torch.int32), tok.to(torch.int32)]


# ---- work --------------------------------------------------------------------------------------------

def work(case):
    op = case["op"]
    if op == "attn":
        q, ctx = _lens(case)
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        vec = d + 4 if case["kv8"] else 2 * d
        kv = sum(q) + sum(ctx)
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(q, ctx))
        return {"bytes": 2 * kv * hkv * vec + 4 * sum(q) * hq * d + 4 * sum(_blocks(n + c) for n, c in zip(q, ctx)),
                "flops": 4 * pairs * hq * d}
    if op == "plan":
        q, ctx = _lens(case)
        rows = sum(q) + case["pad"]
        grown = sum(_blocks(n + c) - _blocks(c) for n, c in zip(q, ctx))
        touched = sum(_blocks(n + c) - c // BLOCK for n, c in zip(q, ctx))
        return {"bytes": 12 * rows + 24 * case["b"] + 4 * touched + 4 * grown, "flops": 4 * rows}
    if op == "append":
        r, hq, hkv, d = (case[k] for k in ("rows", "hq", "hkv", "d"))
        vec = d + 4 if case["kv8"] else 2 * d
        per = 4 * (hq + 2 * hkv) * d + 2 * hq * d + 2 * hkv * vec + 8 + (4 * d if case["rope"] else 0)
        return {"bytes": r * per, "flops": r * (hq + 2 * hkv) * d * 6}
    k = _drafts(case)
    rows = sum(k) + case["b"]
    per = 4 * case["vocab"]
    return {"bytes": rows * per + (case["b"] * per if case["probs"] else 0) + 12 * rows, "flops": 4 * rows * case["vocab"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "plan": _exact_plan, "append": _exact_append, "verify": _exact_verify}[case["op"]](s)


def _exact_attn(s):
    c = s["case"]
    group = c["hq"] // c["hkv"]
    out = torch.zeros((s["q"].shape[0], c["hq"], c["d"]), dtype=torch.float64, device="cuda")
    begin = 0
    for i in range(c["b"]):
        n, ctx = s["q_lens"][i], s["ctx"][i]
        slots = torch.arange(ctx + n, device="cuda")
        blk, off = s["tables"][i].long()[slots // BLOCK], slots % BLOCK
        for h in range(c["hkv"]):
            kk, vv = s["k"][blk, h, off].double(), s["v"][blk, h, off].double()
            if c["kv8"]:
                kk = kk * s["ks"][blk, h, off].double()[:, None]
                vv = vv * s["vs"][blk, h, off].double()[:, None]
            for a in range(0, n, 1024):
                e = min(a + 1024, n)
                q = s["q"][begin + a:begin + e, h * group:(h + 1) * group].double()
                z = torch.einsum("tgd,kd->tgk", q, kk[:ctx + e]) / math.sqrt(c["d"])
                seen = slots[None, :ctx + e] <= (ctx + torch.arange(a, e, device="cuda"))[:, None]
                z = torch.where(seen[:, None], z, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
                out[begin + a:begin + e, h * group:(h + 1) * group] = torch.einsum(
                    "tgk,kd->tgd", torch.softmax(z, -1), vv[:ctx + e])
        begin += n
    return out.reshape(out.shape[0], -1)


def _exact_plan(s):
    rows, width = s["rows"], s["tables"].shape[1]
    q, ctx, have = (s[k].cpu().tolist() for k in ("q_lens", "ctx", "n_blocks"))
    tables, free = s["tables"].cpu().numpy().copy(), s["free"].cpu().numpy()
    at = int(s["cursor"].item())
    cu, pos, slot, seq, kv, held = [0], [], [], [], [], []
    for i, (n, c, h) in enumerate(zip(q, ctx, have)):
        while h < _blocks(c + n):
            tables[i, h] = free[at]
            at, h = at + 1, h + 1
        held.append(h)
        kv.append(c + n)
        cu.append(cu[-1] + n)
        for t in range(c, c + n):
            pos.append(t)
            slot.append(int(tables[i, t // BLOCK]) * BLOCK + t % BLOCK)
            seq.append(i)
    gap = rows - len(pos)
    return [_i32(cu), _i32(kv), _i32(pos + [0] * gap), _i32(slot + [-1] * gap), _i32(seq + [-1] * gap),
            _i32(tables.reshape(-1, width)), _i32(held), _i32([at])]


def _exact_append(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    half = d // 2
    heads = s["qkv"].double().reshape(c["rows"], -1, d)

    def finish(t, weight):
        if weight is not None:
            t = t / torch.sqrt(t.pow(2).sum(-1, keepdim=True) / d + s["eps"]) * weight.double()
        if c["rope"]:
            cs = s["cos_sin"].double()[s["positions"].long()]
            z = torch.complex(t[..., :half], t[..., half:]) * torch.complex(cs[:, None, :half], cs[:, None, half:])
            t = torch.cat([z.real, z.imag], -1)
        return t
    out = [finish(heads[:, :hq], s["qw"])]
    scales = []
    at = s["slots"].long()
    for t in (finish(heads[:, hq:hq + hkv], s["kw"]), heads[:, hq + hkv:]):
        pool = torch.zeros((s["k"].shape[0] * BLOCK, hkv, d), dtype=torch.float64, device="cuda")
        if c["kv8"]:
            sc = torch.clamp(t.abs().max(-1).values / 127, min=1e-8)
            grid = torch.zeros((pool.shape[0], hkv), dtype=torch.float64, device="cuda")
            grid[at] = sc
            scales.append(grid.view(-1, BLOCK, hkv).transpose(1, 2))
            t = torch.round(t / sc[..., None]) * sc[..., None]
        pool[at] = t
        out.append(pool.view(-1, BLOCK, hkv, d).transpose(1, 2))
    return out + scales


def _exact_verify(s):
    k, vocab = s["k"], s["case"]["vocab"]
    acc, tok = [], []
    r0 = 0
    tokens, uni = s["tokens"].cpu().tolist(), s["uniforms"].double().cpu().tolist()
    for i, n in enumerate(k):
        temp = float(s["temps"][i])
        a = 0
        while True:
            row = s["logits"][r0 + a].double()
            if temp == 0.0:
                pick = int(torch.argmax(row))
                if a < n and tokens[r0 + a + 1] == pick:
                    a += 1
                    continue
                break
            p = torch.softmax(row / temp, 0)
            if a == n:
                left = p
            else:
                dr = tokens[r0 + a + 1]
                q = torch.nn.functional.one_hot(torch.tensor(dr, device="cuda"), vocab).double() \
                    if s["probs"] is None else s["probs"][r0 + a].double()
                if uni[r0 + a] * float(q[dr]) < float(p[dr]):
                    a += 1
                    continue
                left = torch.relu(p - q)
                if float(left.sum()) <= 0:
                    left = p
            c = torch.cumsum(left, 0)
            pick = int(torch.searchsorted(c, uni[r0 + n] * c[-1], right=True))
            if pick >= vocab:
                pick = int(torch.nonzero(left)[-1])
            break
        acc.append(a)
        tok.append(pick)
        r0 += n + 1
    return [_i32(acc), _i32(tok)]
