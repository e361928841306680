"""Ragged-batch operators on the GPU against plain 64-bit implementations: the plan, the per-head norm + rotary +
append, the packed causal attention over a paged cache, and the verification of drafts.

Tolerances. A bf16 result is off by half a step, eps/2 = 2^-8 relative at most. The attention rounds its
probabilities to bf16 too: each p_k is off by at most 2^-8 p_k (2^-8 includes nothing else; the fp32 sums and exponentials
add below 2^-16), so out is off by at most 2^-8 sum_k p_k |v_k| + 2^-8 |out| <= 2^-7 sum_k p_k |v_k|, plus the exponential's
argument: scores s up to |s| carry fp32 product sums, 2^-20 |s|. The bound used is 2^-7 * 1.05 * A + 1e-6 with A = sum_k p_k |v_k|."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def K():
    from microgen_b200 import kernels
    return kernels


def i32(a):
    return torch.as_tensor(np.asarray(a, dtype=np.int32), device="cuda")


def errors():
    from microgen_b200 import _lib
    torch.cuda.synchronize()
    return _lib.device_error(torch.cuda.current_stream().cuda_stream, clear=True)


def nblk(n):
    return (n + 15) // 16


# ---------------------------------------------------------------- plan
def plan_oracle(q, ctx, held, tables, free, cursor, rows):
    tables = tables.copy()
    cu, pos, slot, seq, kv, out_held, at = [0], [], [], [], [], [], cursor
    for i, (n, c) in enumerate(zip(q, ctx)):
        h = held[i]
        while h < nblk(c + n):
            tables[i, h] = free[at]
            h, at = h + 1, at + 1
        out_held.append(h)
        kv.append(c + n)
        cu.append(cu[-1] + n)
        for p in range(c, c + n):
            pos.append(p)
            slot.append(tables[i, p // 16] * 16 + p % 16)
            seq.append(i)
    pad = rows - len(pos)
    return cu, kv, pos + [0] * pad, slot + [-1] * pad, seq + [-1] * pad, tables, out_held, at


def plan_case(rng, b, q_max, ctx_max, pad, spare=True):
    q = rng.integers(0, q_max + 1, b)
    ctx = rng.integers(0, ctx_max + 1, b)
    held = np.array([nblk(c) for c in ctx])
    need = np.array([nblk(c + n) for c, n in zip(ctx, q)])
    if spare:
        held = np.minimum(held + rng.integers(0, 3, b), np.maximum(need, held))
    width = int(max(1, need.max(initial=1))) + 2
    total = int(held.sum() + np.maximum(need - held, 0).sum()) + 11
    perm = rng.permutation(total).astype(np.int32)
    tables = np.full((b, width), -7, np.int32)
    at = 0
    for i, h in enumerate(held):
        tables[i, :h] = perm[at:at + h]
        at += h
    cursor = 5
    free = np.concatenate([np.full(cursor, -9, np.int32), perm[at:]])
    return q, ctx, held, tables, free, cursor, int(q.sum()) + pad, total


@pytest.mark.parametrize("b,q_max,ctx_max,pad", [(1, 1, 0, 0), (1, 0, 5, 3), (3, 40, 0, 0), (32, 8, 300, 9), (257, 3, 40, 1),
                                                 (1500, 17, 64, 33), (7, 900, 500, 2000)])
def test_plan_matches_oracle(b, q_max, ctx_max, pad):
    rng = np.random.default_rng(b * 7 + q_max)
    q, ctx, held, tables, free, cursor, rows, total = plan_case(rng, b, q_max, ctx_max, pad)
    plan = K().RaggedPlan(b, rows, tables.shape[1], 8, 2, 64, "cuda")
    td = i32(tables)
    K().ragged_plan(plan, i32(q), i32(ctx), td, total, n_blocks=i32(held), free_blocks=i32(free), cursor=i32([cursor]))
    assert errors()[0] == 0
    want = plan_oracle(q, ctx, held, tables, free, cursor, rows)
    got = [plan.cu_rows, plan.kv_lens, plan.positions, plan.slots, plan.seq_ids, td, plan.n_blocks, plan.cursor]
    for g, w, name in zip(got, want, ("cu", "kv", "pos", "slots", "seq", "tables", "held", "cursor")):
        assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1)), name


def work_list(plan):
    """(entries, merges) of a plan's work area."""
    raw = plan.work.cpu().numpy()
    head = raw[:16].view(np.int32)
    tok_item = 2 * (128 // (plan.hq // plan.hkv))
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    cap = min(plan.max_rows // tok_item + plan.b, plan.max_rows) + max(1, sms // plan.hkv)
    items = raw[64:64 + 32 * cap].view(np.int32).reshape(-1, 8)[:head[0]]
    merges = raw[64 + 32 * cap:].view(np.int32).reshape(-1, 4)[:head[1]]
    return items, merges, tok_item


@pytest.mark.parametrize("b,q_max,ctx_max,hq,hkv", [(1, 1, 40000, 24, 8), (5, 1, 9000, 8, 1), (40, 5, 3000, 24, 8),
                                                    (6, 3000, 100, 12, 12), (300, 60, 50, 16, 1)])
def test_plan_work_list_covers_every_key_once(b, q_max, ctx_max, hq, hkv):
    rng = np.random.default_rng(q_max)
    q, ctx, held, tables, free, cursor, rows, total = plan_case(rng, b, q_max, ctx_max, 3, spare=False)
    q[0], ctx[0] = max(1, q[0] - 1), ctx_max  # (at least one long request; its table has room for it)
    held[0] = nblk(ctx[0])
    tables = np.zeros((b, nblk(ctx_max + q_max) + 2), np.int32)
    plan = K().RaggedPlan(b, rows + 1, tables.shape[1], hq, hkv, 64, "cuda")
    K().ragged_plan(plan, i32(q), i32(ctx), i32(tables), total)
    assert errors()[0] == 0
    items, merges, tok_item = work_list(plan)
    cu = np.concatenate([[0], np.cumsum(q)])
    want = {}
    for i in range(b):
        for j in range((q[i] + tok_item - 1) // tok_item):
            n = min(tok_item, q[i] - j * tok_item)
            want[(i, cu[i] + j * tok_item)] = (n, ctx[i] + j * tok_item, (ctx[i] + j * tok_item + n + 127) // 128)
    seen, slots = {}, {}
    for seq, row0, n, pos0, k0, k1, slot, kv in items:
        n_w, pos_w, tiles = want[(seq, row0)]
        assert (n, pos0, kv) == (n_w, pos_w, pos_w + n_w) and 0 <= k0 < k1 <= tiles
        seen.setdefault((seq, row0), []).append((k0, k1))
        if slot >= 0:
            assert slot not in slots
            slots[slot] = (row0, n)
    assert set(seen) == set(want)
    for key, spans in seen.items():
        spans.sort()
        assert spans[0][0] == 0 and spans[-1][1] == want[key][2]
        assert all(a[1] == c[0] for a, c in zip(spans, spans[1:]))
    split = {k for k, v in seen.items() if len(v) > 1}
    assert len(merges) == len(split)
    for row0, n, slot0, parts in merges:
        assert parts > 1 and all(slots[s] == (row0, n) for s in range(slot0, slot0 + parts))
    assert len(slots) == sum(m[3] for m in merges)


def test_plan_chain_in_place_and_rollback():
    """Steps that feed a plan's own outputs back in, one of them after tokens were taken back: the blocks stay."""
    rng = np.random.default_rng(0)
    b, width, total = 4, 12, 60
    free = rng.permutation(total).astype(np.int32)
    tables = np.zeros((b, width), np.int32)
    plan = K().RaggedPlan(b, 64, width, 8, 2, 64, "cuda")
    td, fd = i32(tables), i32(free)
    ctx, held, cursor = np.zeros(b, int), np.zeros(b, int), 0
    for step, q in enumerate(([20, 1, 0, 33], [1, 16, 3, 1], [5, 5, 5, 5], [17, 1, 1, 1])):
        args = dict(n_blocks=plan.n_blocks, cursor=plan.cursor) if step else {}
        cd = plan.kv_lens if step not in (0, 3) else i32(ctx)
        K().ragged_plan(plan, i32(q), cd, td, total, free_blocks=fd, **args)
        assert errors()[0] == 0
        cu, kv, pos, slot, seq, tables, held, cursor = plan_oracle(q, ctx, held, tables, free, cursor, 64)
        assert np.array_equal(plan.slots.cpu().numpy(), slot) and np.array_equal(td.cpu().numpy(), tables)
        assert plan.n_blocks.tolist() == held and plan.cursor.item() == cursor
        ctx = np.array(kv)
        if step == 2:  # four of each request's last five tokens are taken back
            ctx = ctx - 4
    assert cursor < total


@pytest.mark.parametrize("fault,site", [("neg", 500), ("neg_ctx", 500), ("long", 500), ("held", 502), ("rows", 503),
                                        ("free", 504)])
def test_plan_refuses_impossible_lengths(fault, site):
    b, width = 3, 4
    q, ctx, held, rows, free = [3, 4, 5], [1, 17, 0], [1, 2, 0], 12, np.arange(5)
    if fault == "neg":
        q[1] = -1
    if fault == "neg_ctx":
        ctx[2] = -5
    if fault == "long":
        ctx[0] = 16 * width - 2
    if fault == "held":
        held[1] = 1
    if fault == "rows":
        rows = 11
    if fault == "free":
        free = np.arange(0)
    plan = K().RaggedPlan(b, rows, width, 8, 2, 64, "cuda")
    tables = i32(np.full((b, width), 3))
    K().ragged_plan(plan, i32(q), i32(ctx), tables, 100, n_blocks=i32(held), free_blocks=i32(free))
    code, info = errors()
    assert code == 5 and info == site
    assert plan.cu_rows.tolist() == [0] * (b + 1) and plan.kv_lens.tolist() == [0] * b
    assert (plan.slots == -1).all() and (plan.seq_ids == -1).all() and (tables == 3).all()
    assert plan.n_blocks.tolist() == held and plan.cursor.item() == 0
    assert plan.work[:8].tolist() == [0] * 8  # no work for the attention: it leaves its output alone


@pytest.mark.parametrize("free", [False, True])
def test_plan_refused_without_held_counts_leaves_those_of_the_context(free):
    """``n_blocks`` not given stands for the blocks of ctx: that is what a refused step leaves, and a step after it that takes
    the plan's own counts goes on from there."""
    width, ctx = 6, [33, 0, 16, 1]
    plan = K().RaggedPlan(4, 8, width, 8, 2, 64, "cuda")
    tables = i32(np.arange(4 * width).reshape(4, width))
    kw = dict(free_blocks=i32(np.arange(24, 40))) if free else {}
    K().ragged_plan(plan, i32([3, 4, 5, 6]), i32(ctx), tables, 40, **kw)
    assert errors() == (5, 503)
    assert plan.n_blocks.tolist() == [3, 0, 1, 1]
    K().ragged_plan(plan, i32([9, -1, 0, 0]), i32([33, 0, -7, 1]), tables, 40, **kw)
    assert errors() == (5, 500)
    assert plan.n_blocks.tolist() == [3, 0, 0, 1]
    if free:
        K().ragged_plan(plan, i32([3, 0, 0, 0]), i32([33, 0, 0, 1]), tables, 40, n_blocks=plan.n_blocks, **kw)
        assert errors()[0] == 0 and plan.n_blocks.tolist() == [3, 0, 0, 1]


def test_plan_records_bad_block_ids():
    plan = K().RaggedPlan(2, 4, 2, 8, 2, 64, "cuda")
    K().ragged_plan(plan, i32([2, 2]), i32([0, 15]), i32([[5, 0], [1, 9]]), 9)
    assert errors() == (5, 505)
    assert plan.slots.tolist() == [80, 81, 1 * 16 + 15, -1]


# ---------------------------------------------------------------- append
def append_oracle(qkv, pos, cs, hq, hkv, d, qw, kw, eps):
    x = qkv.astype(np.float64).reshape(len(qkv), -1, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    def norm(t, w):
        return t if w is None else t / np.sqrt((t * t).mean(-1, keepdims=True) + eps) * w
    q, k = norm(q, qw), norm(k, kw)
    if cs is not None:
        c, s = cs[pos][:, None, :d // 2].astype(np.float64), cs[pos][:, None, d // 2:].astype(np.float64)
        def turn(t):
            a, e = t[..., :d // 2], t[..., d // 2:]
            return np.concatenate([a * c - e * s, e * c + a * s], -1)
        q, k = turn(q), turn(k)
    return q, k, v


@pytest.mark.parametrize("hq,hkv,d", [(24, 8, 128), (14, 2, 64), (6, 6, 32), (1, 1, 128), (16, 1, 64)])
@pytest.mark.parametrize("rows,kv8,norm,rope,in16,out16", [
    (1, False, True, True, False, True), (37, True, True, True, False, True), (129, False, False, True, True, False),
    (64, True, False, False, True, True), (5, False, True, False, False, False)])
def test_append_matches_oracle(hq, hkv, d, rows, kv8, norm, rope, in16, out16):
    rng = np.random.default_rng(rows + hq)
    width = (hq + 2 * hkv) * d
    ld = width + 8
    big = torch.from_numpy(rng.standard_normal((rows, ld)).astype(np.float32) * 2).cuda()
    if in16:
        big = big.to(torch.bfloat16)
    qkv = big[:, :width]
    if rows > 3:
        qkv[2] = 0  # a vector of zeros: scale 1e-8, no division by nothing
    blocks = nblk(rows) + 3
    slots = rng.permutation(blocks * 16)[:rows].astype(np.int32)
    if rows > 4:
        slots[[1, rows - 1]] = -1  # padding
    pos = rng.integers(0, 50, rows)
    cs = rng.standard_normal((50, d)).astype(np.float32) if rope else None
    qw = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if norm else None
    kw = (1 + 0.3 * rng.standard_normal(d)).astype(np.float32) if norm else None
    dev = lambda a: None if a is None else torch.from_numpy(a).cuda()
    dt = torch.int8 if kv8 else torch.bfloat16
    kp = torch.full((blocks, hkv, 16, d), 7, dtype=dt, device="cuda")
    vp = torch.full((blocks, hkv, 16, d), 7, dtype=dt, device="cuda")
    sc = {}
    if kv8:
        sc = dict(k_scales=torch.full((blocks, hkv, 16), 0.5, device="cuda"),
                  v_scales=torch.full((blocks, hkv, 16), 0.5, device="cuda"))
    q_out = torch.full((rows, hq, d), 9.0, dtype=torch.bfloat16 if out16 else torch.float32, device="cuda")
    K().norm_rope_kv_append(qkv, i32(pos), dev(cs), i32(slots), hq, hkv, d, kp, vp, q_weight=dev(qw), k_weight=dev(kw),
                            eps=1e-6, q_out=q_out, **sc)
    assert errors()[0] == 0
    q, k, v = append_oracle(qkv.float().cpu().numpy(), pos, cs, hq, hkv, d, qw, kw, 1e-6)
    live = slots >= 0
    # fp32 arithmetic: products and a sum of two, each rounding 2^-24 of terms up to |a c| + |b s|; the norm's sum of d
    # squares, square root and three products: below 2^-20 of the vector's largest value in all
    top = np.abs(np.concatenate([q, k, v], 1)).max(-1, keepdims=True)
    slack = lambda t, i: 2.0 ** -19 * np.maximum(top[:, i], 1e-30)
    def near(got, want, sl, half):
        assert (np.abs(got - want) <= half * np.abs(want) + sl).all(), np.abs(got - want).max()
    qs = 2.0 ** -19 * np.abs(q).max((1, 2), keepdims=True)
    got = q_out.double().cpu().numpy()
    near(got[live], q[live], qs[live], 2.0 ** -8 if out16 else 0)
    assert (got[~live] == 9).all()
    written = np.zeros(blocks * 16, bool)
    written[slots[live]] = True
    for pool, name, want in ((kp, "k_scales", k), (vp, "v_scales", v)):
        rowsp = pool.permute(0, 2, 1, 3).reshape(blocks * 16, hkv, d).double().cpu().numpy()
        w = want[live]
        ws = 2.0 ** -19 * np.abs(w).max((1, 2), keepdims=True) if live.any() else 0
        if kv8:
            s = sc[name].permute(0, 2, 1).reshape(blocks * 16, hkv).double().cpu().numpy()
            s_want = np.maximum(np.abs(w).max(-1) / 127, 1e-8)
            assert (np.abs(s[slots[live]] - s_want) <= 2.0 ** -19 * np.maximum(s_want, np.abs(w).max((1, 2))[:, None] / 127)).all()
            # a code is the nearest whole number of steps: off by half a step, and a tie may fall either way
            near(rowsp[slots[live]] * s[slots[live]][..., None], w, ws + (0.5 + 1e-3) * s_want[..., None], 0)
            assert (s[~written] == 0.5).all()
        else:
            near(rowsp[slots[live]], w, ws, 2.0 ** -8)
        assert (rowsp[~written] == 7).all()


def test_append_matches_the_decode_append():
    """Without norms and with fp32 q the operator stores what rope_kv_append stores."""
    rng = np.random.default_rng(3)
    rows, hq, hkv, d = 19, 24, 8, 128
    qkv = torch.from_numpy(rng.standard_normal((rows, (hq + 2 * hkv) * d)).astype(np.float32)).cuda()
    pos, slots = i32(rng.integers(0, 90, rows)), i32(rng.permutation(4 * 16)[:rows])
    from microgen_b200.engine import rope_table
    cs = rope_table(d, 10000.0, 90).cuda()
    for kv8 in (False, True):
        dt = torch.int8 if kv8 else torch.bfloat16
        pools = [torch.zeros((4, hkv, 16, d), dtype=dt, device="cuda") for _ in range(4)]
        sc = [torch.zeros((4, hkv, 16), device="cuda") for _ in range(4)]
        a = dict(k_scales=sc[0], v_scales=sc[1]) if kv8 else {}
        c = dict(k_scales=sc[2], v_scales=sc[3]) if kv8 else {}
        q0 = K().rope_kv_append(qkv, pos, cs, slots, hq, hkv, d, pools[0], pools[1], **a)
        q1 = K().norm_rope_kv_append(qkv, pos, cs, slots, hq, hkv, d, pools[2], pools[3],
                                     q_out=torch.empty_like(q0), **c)
        torch.testing.assert_close(q1, q0, rtol=0, atol=2.0 ** -20)
        if kv8:
            for i in (0, 1):
                torch.testing.assert_close(sc[i + 2], sc[i], rtol=2.0 ** -20, atol=0)
                assert (pools[i + 2].int() - pools[i].int()).abs().max() <= 1
        else:
            assert all((pools[i + 2].float() - pools[i].float()).abs().max() <= 2.0 ** -7 * pools[i].float().abs().max() for i in (0, 1))
    assert errors()[0] == 0


def test_append_records_bad_positions_and_slots():
    hq, hkv, d = 2, 1, 64
    qkv = torch.ones((2, 4 * d), device="cuda")
    kp = torch.zeros((2, hkv, 16, d), dtype=torch.bfloat16, device="cuda")
    vp = torch.zeros_like(kp)
    cs = torch.ones((5, d), device="cuda")
    K().norm_rope_kv_append(qkv, i32([1, 5]), cs, i32([0, 1]), hq, hkv, d, kp, vp)
    assert errors() == (5, 210)
    K().norm_rope_kv_append(qkv, i32([1, 1]), cs, i32([0, 32]), hq, hkv, d, kp, vp)
    assert errors() == (5, 211)


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("pos", [-1, 5, 2 ** 31 - 1])
def test_append_writes_nothing_of_a_row_outside_the_table(pos, kv8):
    hq, hkv, d = 2, 1, 64
    dt = torch.int8 if kv8 else torch.bfloat16
    kp, vp = (torch.full((2, hkv, 16, d), 7, dtype=dt, device="cuda") for _ in range(2))
    sc = dict(k_scales=torch.full((2, hkv, 16), 7.0, device="cuda"), v_scales=torch.full((2, hkv, 16), 7.0, device="cuda")) if kv8 else {}
    q = torch.full((3, hq, d), 7.0, dtype=torch.bfloat16, device="cuda")
    K().norm_rope_kv_append(torch.ones((3, 4 * d), device="cuda"), i32([1, pos, 4]), torch.ones((5, d), device="cuda"), i32([3, 4, 5]),
                            hq, hkv, d, kp, vp, q_out=q, **sc)
    assert errors() == (5, 210)
    for t in (kp[0, 0], vp[0, 0], *(s[0, 0] for s in sc.values())):
        assert (t[4] == 7).all() and (t[3] != 7).any() and (t[5] != 7).any()
    assert (q[1] == 7).all() and (q[0] != 7).all() and (q[2] != 7).all()


@pytest.mark.parametrize("hq,hkv,d", [(14, 2, 64), (6, 6, 32), (3, 1, 128)])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_append_int8_keeps_what_is_not_a_number(hq, hkv, d, bad):
    """A vector with an infinity or NaN reads back as NaN; the vectors beside it are stored as without it."""
    rng = np.random.default_rng(d)
    rows = 9
    x = torch.from_numpy(rng.standard_normal((rows, (hq + 2 * hkv) * d)).astype(np.float32)).cuda()
    slots = i32(rng.permutation(32)[:rows])

    def run(qkv):
        kp, vp = (torch.zeros((2, hkv, 16, d), dtype=torch.int8, device="cuda") for _ in range(2))
        ks, vs = (torch.zeros((2, hkv, 16), device="cuda") for _ in range(2))
        K().norm_rope_kv_append(qkv, None, None, slots, hq, hkv, d, kp, vp, k_scales=ks, v_scales=vs)
        at = lambda p, s: (p.float() * s[..., None]).transpose(1, 2).reshape(32, hkv, d)[slots.long()]
        return torch.cat([at(kp, ks), at(vp, vs)], 1)  # [rows, 2 hkv, d]: K's vectors, then V's

    clean = run(x)
    hit = torch.zeros((rows, 2 * hkv), dtype=torch.bool, device="cuda")
    heads = x.view(rows, -1, d)
    for r, h, c in ((1, 0, 0), (1, 2 * hkv - 1, d - 1), (4, hkv, d // 2), (8, hkv - 1, 5)):
        heads[r, hq + h, c] = bad
        hit[r, h] = True
    got = run(x)
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])
    assert errors()[0] == 0


# ---------------------------------------------------------------- attention
class Case:
    def __init__(self, q, ctx, hq, hkv, d, kv8=False, seed=0, pad=0, spread=1.0):
        rng = np.random.default_rng(seed)
        self.q_lens, self.ctx, self.hq, self.hkv, self.d, self.kv8 = list(q), list(ctx), hq, hkv, d, kv8
        need = [nblk(a + c) for a, c in zip(q, ctx)]
        self.blocks = sum(need) + 3
        perm = rng.permutation(self.blocks).astype(np.int32)
        self.tables = np.zeros((len(q), max(need + [1])), np.int32)
        at = 0
        for i, n in enumerate(need):
            self.tables[i, :n] = perm[at:at + n]
            at += n
        g = torch.Generator(device="cuda").manual_seed(seed)
        rows = sum(q) + pad
        self.q = (torch.randn((rows, hq, d), generator=g, device="cuda") * spread).to(torch.bfloat16)
        shape = (self.blocks, hkv, 16, d)
        k, v = torch.randn(shape, generator=g, device="cuda"), torch.randn(shape, generator=g, device="cuda")
        self.sc = {}
        if kv8:
            sk, sv = k.abs().amax(-1) / 127, v.abs().amax(-1) / 127
            self.k = torch.round(k / sk[..., None]).to(torch.int8)
            self.v = torch.round(v / sv[..., None]).to(torch.int8)
            self.sc = dict(k_scales=sk.contiguous(), v_scales=sv.contiguous())
        else:
            self.k, self.v = k.to(torch.bfloat16), v.to(torch.bfloat16)
        self.scale = 1 / math.sqrt(d)
        self.plan = K().RaggedPlan(len(q), rows, self.tables.shape[1], hq, hkv, d, "cuda")
        self.td = i32(self.tables)

    def fill(self):
        K().ragged_plan(self.plan, i32(self.q_lens), i32(self.ctx), self.td, self.blocks)
        return self

    def run(self, **kw):
        return K().ragged_attn(self.q, self.k, self.v, self.plan, self.scale, **self.sc, **kw)

    def oracle(self):
        """(out, sum_k p_k |v_k|) fp64 [rows, hq, d] of the live rows."""
        outs, mags = [], []
        kf, vf = self.k.double(), self.v.double()
        if self.kv8:
            kf, vf = kf * self.sc["k_scales"].double()[..., None], vf * self.sc["v_scales"].double()[..., None]
        r = 0
        for i, (n, c) in enumerate(zip(self.q_lens, self.ctx)):
            ids = self.td[i, :nblk(c + n)].long()
            kk = kf[ids].transpose(1, 2).reshape(-1, self.hkv, self.d)[:c + n]
            vv = vf[ids].transpose(1, 2).reshape(-1, self.hkv, self.d)[:c + n]
            q = self.q[r:r + n].double().view(n, self.hkv, self.hq // self.hkv, self.d)
            s = torch.einsum("nhgd,khd->hgnk", q, kk) * self.scale
            see = torch.arange(c + n, device="cuda")[None] <= c + torch.arange(n, device="cuda")[:, None]
            p = torch.softmax(s.masked_fill(~see, -math.inf), -1)
            outs.append(torch.einsum("hgnk,khd->nhgd", p, vv).reshape(n, self.hq, self.d))
            mags.append(torch.einsum("hgnk,khd->nhgd", p, vv.abs()).reshape(n, self.hq, self.d))
            r += n
        return torch.cat(outs), torch.cat(mags)


def check_attn(case, out, rows=None):
    want, mag = case.oracle()
    got = out[:want.shape[0]].double().view_as(want)
    err = (got - want).abs()
    bound = 2.0 ** -7 * 1.05 * mag + 1e-6
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"max err {err.max().item():.3e}, {int((err > bound).sum())} of {err.numel()} outside"
    assert errors()[0] == 0


HEADS = [(24, 8, 128), (14, 2, 64), (6, 6, 32), (12, 12, 64), (16, 1, 64), (3, 1, 128)]


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("q,ctx", [([1], [0]), ([1], [15]), ([1], [127]), ([1], [128]), ([5], [300]),
                                   ([7, 0, 130, 1, 16], [0, 5, 77, 1000, 16])])
def test_attention_small(hq, hkv, d, q, ctx, kv8):
    c = Case(q, ctx, hq, hkv, d, kv8, seed=len(q) + ctx[0]).fill()
    check_attn(c, c.run())


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_attention_prompts_and_mixtures(hq, hkv, d, kv8):
    c = Case([300, 1, 129, 513, 2, 85, 84, 83], [0, 700, 0, 250, 33, 0, 128, 1], hq, hkv, d, kv8, seed=5).fill()
    check_attn(c, c.run())


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("hq,hkv,d", [(24, 8, 128), (16, 1, 64), (6, 6, 32)])
@pytest.mark.parametrize("q,ctx", [([1], [9000]), ([1, 1, 3], [20000, 17, 5000]), ([200], [6000])])
def test_attention_split_over_keys(hq, hkv, d, q, ctx, kv8):
    c = Case(q, ctx, hq, hkv, d, kv8, seed=9).fill()
    assert work_list(c.plan)[1].shape[0] > 0  # the plan splits these
    check_attn(c, c.run())


def test_attention_large_scores():
    """Scores in the hundreds: maxima that grow along the keys, so that the output is rescaled; nearly one-hot rows."""
    c = Case([200, 1], [900, 3000], 24, 8, 128, seed=2, spread=12.0).fill()
    check_attn(c, c.run())


def test_attention_leaves_rows_behind_the_batch():
    c = Case([3, 60], [10, 0], 14, 2, 64, seed=4, pad=90).fill()
    out = torch.full((c.q.shape[0], 14 * 64), 5.0, dtype=torch.bfloat16, device="cuda")
    got = c.run(out=out)
    check_attn(c, got)
    assert (out[63:] == 5).all()


@pytest.mark.parametrize("kv8", [False, True])
def test_attention_ignores_what_a_row_may_not_see(kv8):
    """NaN and infinities behind the last token, and in tokens that earlier rows of the same tile may not see."""
    c = Case([150, 20, 1], [0, 100, 260], 24, 8, 128, kv8, seed=6).fill()
    clean = c.run().clone()
    for i, (n, x) in enumerate(zip(c.q_lens, c.ctx)):  # the rest of every last block
        blk, off = c.tables[i, (n + x - 1) // 16], (n + x - 1) % 16 + 1
        if off < 16:
            if kv8:
                for s in c.sc.values():
                    s[blk, :, off:] = math.nan
            else:
                c.k[blk, :, off:] = math.nan
                c.v[blk, :, off:] = math.inf
    spare = np.setdiff1d(np.arange(c.blocks), c.tables.reshape(-1))
    if not kv8:
        c.k[spare], c.v[spare] = math.nan, math.nan
    assert torch.equal(c.run(), clean)
    # token 100 of request 0: rows before it must not change, rows from it on see it
    blk, off = c.tables[0, 100 // 16], 100 % 16
    for bad in (math.nan, math.inf):
        if kv8:
            c.sc["v_scales"][blk, 2, off] = bad
        else:
            c.v[blk, 2, off, 17] = bad
        got = c.run().view(-1, 8, 3, 128)
        ref = clean.view(-1, 8, 3, 128)
        assert torch.equal(got[150:], ref[150:])
        near = (got[:100].double() - ref[:100].double()).abs() <= 2.0 ** -6 * ref[:100].double().abs().clamp(min=0.25)
        assert near.all()
        assert torch.equal(got[:, [0, 1, 3, 4, 5, 6, 7]], ref[:, [0, 1, 3, 4, 5, 6, 7]])
        seen = got[100:150, 2]
        if not kv8:
            assert not torch.isfinite(seen[..., 17]).any()
            rest = [x for x in range(128) if x != 17]
            assert torch.isfinite(seen[..., rest]).all()
            near = (seen[..., rest].double() - ref[100:150, 2][..., rest].double()).abs() <= 2.0 ** -6 * ref[100:150, 2][..., rest].double().abs().clamp(min=0.25)
            assert near.all()
        else:
            assert not torch.isfinite(seen).any()
    assert errors()[0] == 0


@pytest.mark.parametrize("hq,hkv,d", [(24, 8, 128), (14, 2, 64), (6, 6, 32)])
@pytest.mark.parametrize("b,q,ctx", [(40, (10, 40), (0, 0)), (64, (5, 5), (0, 100)), (24, (90, 300), (0, 60))])
def test_attention_ignores_masked_values_of_many_pieces(hq, hkv, d, b, q, ctx):
    """An infinity or NaN in a late token's V of nearly every request and K/V head, in a column of its own: a CTA has several
    such pieces one behind another, and what it found in one must not be taken for, or lost in, the next."""
    rng = np.random.default_rng(b)
    c = Case(rng.integers(q[0], q[1] + 1, b), rng.integers(ctx[0], ctx[1] + 1, b), hq, hkv, d, seed=b).fill()
    clean = c.run().clone()
    want, mag = c.oracle()  # of the clean values
    bad_row = torch.zeros_like(want, dtype=torch.bool)
    same = torch.zeros(want.shape[0], dtype=torch.bool, device="cuda")
    r = 0
    for i, (n, x) in enumerate(zip(c.q_lens, c.ctx)):
        t = int(rng.integers(n // 2 + 1, n))
        if i % 5 == 4:
            same[r:r + n] = True
        else:
            blk, off = c.tables[i, (x + t) // 16], (x + t) % 16
            for h in range(hkv):
                col = (7 * i + 13 * h) % d
                c.v[blk, h, off, col] = (math.nan, math.inf, -math.inf)[(i + h) % 3]
                bad_row[r + t:r + n, h * (hq // hkv):(h + 1) * (hq // hkv), col] = True
        r += n
    bound = 2.0 ** -7 * 1.05 * mag + 1e-6
    for _ in range(6):
        out = c.run()
        assert torch.equal(out[same], clean[same])
        got = out.double().view_as(want)
        assert not torch.isfinite(got[bad_row]).any()
        assert ((got - want).abs() <= bound)[~bad_row].all()
    assert errors()[0] == 0


NAN_CASES = [([1], [100]), ([1], [128]), ([1], [300]), ([1], [20000]), ([60], [0]), ([200], [100]), ([40, 1], [9000, 7])]


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("q,ctx", NAN_CASES)
def test_attention_gives_nan_for_a_nan_that_a_row_sees(q, ctx, kv8):
    """A NaN in a query, or in the K of a key: NaN in the rows that meet it and in no others, in every form of an item (one
    row tile or two, whose keys one warpgroup takes or both, split along the keys or not)."""
    def check(c, bad):
        want, mag = c.oracle()
        got = c.run().double().view_as(want)
        assert torch.isnan(got[bad]).all()
        assert ((got - want).abs() <= 2.0 ** -7 * 1.05 * mag + 1e-6)[~bad].all()
        assert errors()[0] == 0

    c = Case(q, ctx, 24, 8, 128, kv8, seed=1).fill()
    bad = torch.zeros((sum(q), 24), dtype=torch.bool, device="cuda")
    for r in {0, q[0] // 2, q[0] - 1}:
        c.q[r, 5 + r % 7, 7] = math.nan
        bad[r, 5 + r % 7] = True
    check(c, bad)
    c = Case(q, ctx, 24, 8, 128, kv8, seed=2).fill()
    t = q[0] // 2  # the new token whose K holds it
    at = (c.tables[0, (ctx[0] + t) // 16], 2, (ctx[0] + t) % 16)
    if kv8:
        c.sc["k_scales"][at] = math.nan
    else:
        c.k[at][3] = math.nan
    bad = torch.zeros((sum(q), 24), dtype=torch.bool, device="cuda")
    bad[t:q[0], 6:9] = True
    check(c, bad)


@pytest.mark.parametrize("q,ctx", NAN_CASES)
def test_attention_gives_nan_where_every_score_is_minus_infinity(q, ctx):
    c = Case(q, ctx, 24, 8, 128, seed=3).fill()
    c.q[:, :3] = 1.0
    c.k[:, 0] = 1.0
    c.k[:, 0, :, 3] = -math.inf
    got = c.run().view(-1, 24, 128)
    assert torch.isnan(got[:, :3]).all() and torch.isfinite(got[:, 3:]).all()
    assert errors()[0] == 0


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("q,ctx,big,at", [([1], [255], 3, 200), ([1], [255], 200, 3), ([1], [20000], 5, 15000), ([1], [20000], 15000, 5),
                                          ([200], [9000], 7, 6000), ([60], [0], 3, 20), ([120], [0], 3, 50)])
def test_attention_keeps_a_value_whose_weight_is_zero_in_32_bits(q, ctx, big, at, bad, kv8):
    """One key takes all the weight; another, in a tile or part of its own, holds an infinity or NaN in V: zero times it is NaN, as
    in the plain form, although the part's whole weight is zero when states are merged."""
    hq, hkv, d = 24, 8, 128
    c = Case(q, ctx, hq, hkv, d, kv8, seed=4).fill()
    place = lambda p: (c.tables[0, p // 16], 2, p % 16)
    c.q[:] = 1.0
    c.k.zero_()
    if kv8:  # 16 in every place: 181 above the other scores
        c.k[place(big)] = 127
        c.sc["k_scales"][place(big)] = 16.0 / 127
        c.sc["v_scales"][place(at)] = bad
    else:
        c.k[place(big)] = 16.0
        c.v[place(at)][5] = bad
    out = c.run().view(-1, hq, d)
    assert errors()[0] == 0
    first = max(0, at - ctx[0])  # the first new token that sees it
    cols = slice(None) if kv8 else slice(5, 6)
    assert not torch.isfinite(out[first:, 6:9, cols]).any()
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[first:, 6:9, cols] = False
    assert torch.isfinite(out[rest]).all()


@pytest.mark.parametrize("kv8", [False, True])
@pytest.mark.parametrize("q,ctx,hq,hkv,d,req,at", [([244, 296, 69], [49, 102, 142], 8, 8, 128, 1, 287), ([40], [630], 12, 12, 64, 0, 592),
                                                   ([34, 37], [150, 625], 12, 12, 64, 1, 607)])
def test_attention_keeps_a_nan_in_a_part_whose_last_tile_a_row_does_not_see(q, ctx, hq, hkv, d, req, at, kv8):
    """A part of a split item ends in a tile that lies behind some of its rows, and the tile before holds a NaN in K: the part's
    two states are a NaN and an empty one, and the merge of the parts must not take what comes of them for empty."""
    c = Case(q, ctx, hq, hkv, d, kv8, seed=5).fill()
    assert work_list(c.plan)[1].shape[0] > 0  # the plan splits these
    want, mag = c.oracle()
    place = (c.tables[req, at // 16], 1, at % 16)
    if kv8:
        c.sc["k_scales"][place] = math.nan
    else:
        c.k[place][0] = math.nan
    bad = torch.zeros(want.shape[:2], dtype=torch.bool, device="cuda")
    start = sum(q[:req])
    bad[start + max(0, at - ctx[req]):start + q[req], hq // hkv:2 * (hq // hkv)] = True
    got = c.run().double().view_as(want)
    assert torch.isnan(got[bad]).all()
    assert ((got - want).abs() <= 2.0 ** -7 * 1.05 * mag + 1e-6)[~bad].all()
    assert errors()[0] == 0


def test_attention_matches_the_decode_kernel():
    """Single tokens: the operator gives what paged_decode_attn gives (which rounds q * scale to bf16)."""
    c = Case([1] * 6, [3, 63, 500, 1999, 0, 128], 24, 8, 128, seed=8).fill()
    got = c.run().double()
    ctx = i32([x + 1 for x in c.ctx])
    ref = K().paged_decode_attn(c.q.float(), c.k, c.v, c.td, ctx, c.scale).double()
    assert ((got - ref).abs() <= 1e-2 + 2e-2 * ref.abs()).all()


def test_attention_repeats_exactly_and_on_another_stream():
    c = Case([1, 40, 1], [15000, 3000, 9], 24, 8, 128, seed=10).fill()
    first = c.run()
    for _ in range(3):
        assert torch.equal(c.run(), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = c.run()
    s.synchronize()
    assert torch.equal(other, first)


def test_attention_and_plan_in_a_graph():
    """A captured step replayed with other lengths: the plan and the attention follow the device's numbers."""
    c = Case([40, 3, 1], [0, 200, 700], 14, 2, 64, seed=12)
    q_lens, ctx = i32(c.q_lens), i32(c.ctx)
    out = torch.zeros((c.q.shape[0], 14 * 64), dtype=torch.bfloat16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K().ragged_plan(c.plan, q_lens, ctx, c.td, c.blocks)
        c.run(out=out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K().ragged_plan(c.plan, q_lens, ctx, c.td, c.blocks)
        c.run(out=out)
    for ql, cx in (([40, 3, 1], [0, 200, 700]), ([10, 30, 4], [30, 100, 3]), ([0, 0, 44], [0, 0, 650]), ([1, 1, 1], [5, 6, 7])):
        q_lens.copy_(i32(ql))
        ctx.copy_(i32(cx))
        out.fill_(3.0)
        g.replay()
        c.q_lens, c.ctx = ql, cx
        check_attn(c, out)
        assert (out[sum(ql):] == 3).all()


def test_two_steps_at_once_and_the_most_requests():
    """Steps on two streams, each with a plan of its own; and a plan of as many requests as there may be."""
    cases = [Case([300, 1, 70], [0, 9000, 500], 24, 8, 128, seed=21), Case([1, 1, 5], [12000, 40, 3000], 24, 8, 128, seed=22)]
    want = [c.fill().run() for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(8):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                c.fill()
                got[i].append(c.run())
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)
    c = Case([1] * 8192, [i % 3 for i in range(8192)], 3, 1, 32, seed=23).fill()
    check_attn(c, c.run())


def test_attention_refuses_wrong_arguments():
    c = Case([4], [0], 14, 2, 64)
    with pytest.raises(ValueError):
        c.run()  # not planned
    c.fill()
    for kw in (dict(q=c.q.float()), dict(q=c.q[:, :13]), dict(k=c.k[:, :1]), dict(k=c.k.to(torch.float16)), dict(scale=0.0),
               dict(scale=-1.0), dict(v=c.v.cpu()), dict(out=torch.empty(3, 14 * 64, dtype=torch.bfloat16, device="cuda")),
               dict(k_scales=torch.ones(c.blocks, 2, 16, device="cuda"))):
        a = dict(q=c.q, k=c.k, v=c.v, scale=c.scale)
        a.update({k: v for k, v in kw.items() if k in a})
        rest = {k: v for k, v in kw.items() if k not in a}
        with pytest.raises((ValueError, TypeError)):
            K().ragged_attn(a["q"], a["k"], a["v"], c.plan, a["scale"], **rest)


def test_attention_records_a_plan_for_more_rows():
    c = Case([9, 9], [0, 0], 14, 2, 64).fill()
    out = torch.full((10, 14 * 64), 2.0, dtype=torch.bfloat16, device="cuda")
    K().ragged_attn(c.q[:10].contiguous(), c.k, c.v, c.plan, c.scale, out=out)
    assert errors() == (5, 510)


@pytest.mark.parametrize("other", [dict(max_rows=700), dict(b=3), dict(hq=16, hkv=16), dict(hq=48), dict(max_blocks=700)])
def test_attention_records_a_plan_for_other_sizes(other):
    """A work area that was planned for other sizes has its list elsewhere: it is recorded and nothing of it is run, neither
    by the attention nor by the merge of split items."""
    from microgen_b200 import _lib
    c = Case([1, 40], [9000, 500], 24, 8, 64, seed=1).fill()
    assert work_list(c.plan)[1].shape[0] > 0
    p = c.plan
    a = dict(max_rows=p.max_rows, b=p.b, hq=p.hq, hkv=p.hkv, max_blocks=p.max_blocks)
    a.update(other)
    q = torch.zeros((41, a["hq"], 64), dtype=torch.bfloat16, device="cuda")
    out = torch.full((41, a["hq"] * 64), 2.0, dtype=torch.bfloat16, device="cuda")
    pool = torch.zeros((c.blocks, a["hkv"], 16, 64), dtype=torch.bfloat16, device="cuda")
    tables = torch.zeros((a["b"], a["max_blocks"]), dtype=torch.int32, device="cuda")
    ws = K().RaggedPlan(a["b"], a["max_rows"], a["max_blocks"], a["hq"], a["hkv"], 64, "cuda").workspace
    _lib.call("mg_ragged_attn", q.data_ptr(), 41, pool.data_ptr(), pool.data_ptr(), None, None, c.blocks, tables.data_ptr(),
              a["max_blocks"], a["b"], a["max_rows"], a["hq"], a["hkv"], 64, 0.125, p.work.data_ptr(), out.data_ptr(),
              ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream)
    assert errors() == (5, 510)
    assert (out == 2).all()
    check_attn(c, c.run())


def test_an_empty_plan_gives_the_attention_nothing_to_do():
    c = Case([4, 9], [3, 100], 14, 2, 64)
    c.q_lens[0] = 100  # one length alone is more than the plan's rows
    c.fill()
    assert errors() == (5, 500)
    out = torch.full((13, 14 * 64), 2.0, dtype=torch.bfloat16, device="cuda")
    c.run(out=out)
    assert errors()[0] == 0 and (out == 2).all()


# ---------------------------------------------------------------- verification
def verify_oracle(logits, tokens, cu, u, probs, temps):
    lg = logits.double().cpu().numpy()
    acc, nxt = [], []
    for i in range(len(cu) - 1):
        r0, n = cu[i], cu[i + 1] - cu[i] - 1
        if n < 0:
            acc.append(0)
            nxt.append(-1)
            continue
        t = 1.0 if temps is None else float(np.float32(temps[i]))
        a = 0
        while True:
            row = lg[r0 + a]
            if t == 0:
                pick = int(np.argmax(row))
                if a < n and tokens[r0 + a + 1] == pick:
                    a += 1
                    continue
                break
            z = row / t
            p = np.exp(z - z.max())
            p /= p.sum()
            w = p
            if a < n:
                d = tokens[r0 + a + 1]
                q = np.zeros_like(p)
                if probs is None:
                    q[d] = 1.0
                else:
                    q = probs[r0 + a].double().cpu().numpy()
                if float(u[r0 + a]) * q[d] < p[d]:
                    a += 1
                    continue
                w = np.maximum(p - q, 0)
                if w.sum() <= 0:
                    w = p
            c = np.cumsum(w)
            pick = int(np.searchsorted(c, float(u[r0 + n]) * c[-1], side="right"))
            if pick >= len(c):
                pick = int(np.nonzero(w)[0][-1])
            break
        acc.append(a)
        nxt.append(pick)
    return acc, nxt


def verify_case(ks, vocab, probs, seed, temps=None, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    cu = np.concatenate([[0], np.cumsum([k + 1 for k in ks])]).astype(np.int32)
    rows = int(cu[-1])
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * spread
    q = torch.softmax(logits + 0.5 * torch.randn((rows, vocab), generator=g, device="cuda"), -1)
    drawn = torch.multinomial(q, 1, generator=g)[:, 0].cpu().numpy()
    best = logits.argmax(-1).cpu().numpy()
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    for i, k in enumerate(ks):
        for j in range(k):
            tokens[cu[i] + j + 1] = best[cu[i] + j] if (temps is not None and temps[i] == 0) or rng.random() < 0.3 else drawn[cu[i] + j]
    u = torch.rand(rows, generator=g, device="cuda")
    return logits, tokens, cu, u, q if probs else None


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("vocab", [1, 3, 32, 33, 1000, 4097, 50257, 128256])
def test_verify_matches_oracle(vocab, probs):
    ks = [0, 1, 4, 8, 2, 3, 5, 0, 19]
    for seed in range(3):
        temps = np.array([1.0, 0.7, 0.0, 1.3, 1.0, 0.05, 0.9, 0.0, 1.0], np.float32) if seed else None
        logits, tokens, cu, u, q = verify_case(ks, vocab, probs, seed + vocab, temps)
        got = K().verify_drafts(logits, i32(tokens), i32(cu), u, draft_probs=q,
                                temperatures=None if temps is None else torch.from_numpy(temps).cuda())
        want = verify_oracle(logits, tokens, cu, u.cpu().numpy(), q, temps)
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert errors()[0] == 0


def test_verify_in_a_graph_and_on_two_streams():
    """A captured verification replayed on other numbers, and two of them at once in workspaces of their own."""
    cases = [verify_case([3, 0, 6, 1], 50257, probs, 30 + int(probs)) for probs in (False, True)]
    tok, cu = [i32(c[1]) for c in cases], [i32(c[2]) for c in cases]

    def run(i, **kw):
        return K().verify_drafts(cases[i][0], tok[i], cu[i], cases[i][3], draft_probs=cases[i][4], **kw)

    def want(i):
        lg, _, c, u, q = cases[i]
        return verify_oracle(lg, tok[i].cpu().numpy(), c, u.cpu().numpy(), q, None)

    for i in range(2):
        acc, nxt = i32([0] * 4), i32([0] * 4)
        ws = torch.empty(K().verify_workspace_bytes(cases[i][0].shape[0], 50257, 4), dtype=torch.uint8, device="cuda")
        run(i, accepted=acc, next_tokens=nxt, workspace=ws)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run(i, accepted=acc, next_tokens=nxt, workspace=ws)
        for seed in (41, 42, 43):
            new = verify_case([3, 0, 6, 1], 50257, bool(i), seed + 10 * i)
            cases[i][0].copy_(new[0])
            tok[i].copy_(i32(new[1]))
            cases[i][3].copy_(new[3])
            if i:
                cases[i][4].copy_(new[4])
            ws.fill_(255)  # nothing is kept in it from one call to the next
            g.replay()
            assert [acc.tolist(), nxt.tolist()] == list(want(i))
    expect = [want(i) for i in range(2)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(i))
    torch.cuda.synchronize()
    for e, g in zip(expect, got):
        assert all([a.tolist(), n.tolist()] == list(e) for a, n in g)
    assert errors()[0] == 0


def test_verify_strided_and_empty_requests():
    logits, tokens, cu, u, q = verify_case([3, 2, 1], 777, True, 5)
    wide = torch.full((logits.shape[0], 801), 50.0, device="cuda")
    wide[:, 3:780] = logits
    view = wide[:, 3:780]  # rows that start off a 16-byte boundary
    cu2 = np.array([cu[0], cu[1], cu[1], cu[2], cu[3], cu[3]], np.int32)  # requests without rows
    got = K().verify_drafts(view, i32(tokens), i32(cu2), u, draft_probs=q)
    want = verify_oracle(logits, tokens, cu2, u.cpu().numpy(), q, None)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    none = K().verify_drafts(view[:0], i32([]), i32([0, 0]), u[:0])
    assert none[0].tolist() == [0] and none[1].tolist() == [-1]
    assert errors()[0] == 0


def test_verify_same_distributions_accept_and_fall_back():
    """q = p: every draft is accepted for u < 1; and where a draft with q(d) = 0 = p(d) is turned down although the
    distributions agree everywhere, the token comes from p."""
    vocab = 64
    logits = torch.full((3, vocab), -math.inf, device="cuda")
    logits[:, :2] = 0.0
    q = torch.softmax(logits, -1)
    tokens = i32([0, 0, 40])  # second draft: a token that neither gives any probability
    u = torch.tensor([0.999, 0.0, 0.75], device="cuda")
    acc, nxt = K().verify_drafts(logits, tokens, i32([0, 3]), u, draft_probs=q)
    assert acc.tolist() == [1] and nxt.tolist() == [1]
    assert errors()[0] == 0


def test_verify_distribution_is_the_targets():
    """Over many draws the first token's frequencies are the target's, whatever the draft proposes."""
    vocab, n = 12, 20000
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.softmax(torch.randn(vocab, generator=g, device="cuda"), 0)
    q = torch.softmax(torch.randn(vocab, generator=g, device="cuda"), 0)
    logits = p.log().repeat(2 * n, 1)
    d = torch.multinomial(q.repeat(n, 1), 1, generator=g)[:, 0].to(torch.int32)
    tokens = torch.stack([torch.zeros_like(d), d], 1).reshape(-1).contiguous()
    u = torch.rand(2 * n, generator=g, device="cuda")
    cu = torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda")
    first = []
    for lo in range(0, n, 10000):  # (rows are a grid dimension of at most 65535)
        s = slice(2 * lo, 2 * (lo + 10000))
        acc, nxt = K().verify_drafts(logits[s], tokens[s], cu[:10001], u[s], draft_probs=q.repeat(20000, 1))
        first.append(torch.where(acc > 0, d[lo:lo + 10000], nxt))
    freq = torch.bincount(torch.cat(first).long(), minlength=vocab).double() / n
    # five standard deviations of a binomial proportion
    assert ((freq - p.double()).abs() <= 5 * (p.double() * (1 - p.double()) / n).sqrt()).all()
    assert errors()[0] == 0


@pytest.mark.parametrize("what,site", [("nan", 604), ("inf", 604), ("empty", 604), ("temp", 602), ("token", 603), ("cu", 601)])
def test_verify_records_what_it_cannot_answer(what, site):
    logits, tokens, cu, u, _ = verify_case([2, 2], 100, False, 3)
    temps = torch.ones(2, device="cuda")
    tokens = tokens.copy()
    if what == "nan":
        logits[0, 50] = math.nan
    if what == "inf":
        logits[0, 50] = math.inf
    if what == "empty":
        logits[0] = -math.inf
    if what == "temp":
        temps[0] = -1.0
    if what == "token":
        tokens[1] = 100
    if what == "cu":
        cu = np.array([0, 3, 7], np.int32)
    acc, nxt = K().verify_drafts(logits, i32(tokens), i32(cu), u, temperatures=temps)
    assert errors() == (5, site)
    bad = 1 if what == "cu" else 0
    assert acc[bad].item() == 0
    assert nxt[bad].item() == -1 if what != "token" else 0 <= nxt[bad].item() < 100
    ok = 1 - bad
    want = verify_oracle(logits.nan_to_num(0, 0, -50), tokens.clip(0, 99), [0, 3, 6], u.cpu().numpy(), None, None)
    assert (acc[ok].item(), nxt[ok].item()) == (want[0][ok], want[1][ok])


@pytest.mark.parametrize("t", [-1.0, math.nan])
def test_verify_bad_temperature_beside_a_bad_draft(t):
    """Two things wrong with one request: without a temperature there is no answer, whatever its drafts are."""
    logits, tokens, cu, u, _ = verify_case([2, 2], 100, False, 3)
    tokens = tokens.copy()
    tokens[1] = 100
    temps = torch.tensor([t, 1.0], device="cuda")
    acc, nxt = K().verify_drafts(logits, i32(tokens), i32(cu), u, temperatures=temps)
    assert errors() == (5, 602)
    want = verify_oracle(logits, tokens.clip(0, 99), cu, u.cpu().numpy(), None, None)
    assert (acc.tolist(), nxt.tolist()) == ([0, want[0][1]], [-1, want[1][1]])


def test_verify_invalid_draft_behind_the_stop():
    """A drafted token outside the vocabulary behind the place where the request stops is recorded, and changes nothing:
    the token that was turned down is still not drawn again."""
    vocab, n = 4, 400
    logits = torch.zeros((3 * n, vocab), device="cuda")
    tokens = i32([0, 2, 9] * n)  # the first draft is turned down (u = 1 - 2^-24 > p), the second is no token
    u = torch.rand(3 * n, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")
    u[0::3] = 1 - 2.0 ** -24
    acc, nxt = K().verify_drafts(logits, tokens, torch.arange(0, 3 * n + 1, 3, dtype=torch.int32, device="cuda"), u)
    assert errors() == (5, 603)
    assert (acc == 0).all() and (nxt != 2).all() and set(nxt.tolist()) == {0, 1, 3}


def test_verify_at_the_edges_of_the_uniform_numbers():
    """u = 0 draws the first index with any weight, u = 1 (or a little more) the last."""
    logits = torch.full((2, 1000), -math.inf, device="cuda")
    logits[:, 17:900:3] = 0.5
    for u, want in ((0.0, 17), (1.0, 17 + 3 * 294), (1.5, 17 + 3 * 294)):
        _, nxt = K().verify_drafts(logits, i32([1, 1]), i32([0, 1, 2]), torch.full((2,), u, device="cuda"))
        assert nxt.tolist() == [want, want]
    assert errors()[0] == 0


def test_verify_refuses_outputs_over_inputs():
    logits, tokens, cu, u, _ = verify_case([2, 2], 100, False, 3)
    tokens, cu = i32(tokens), i32(cu)
    buf = i32(np.zeros(5))
    from microgen_b200 import _lib
    for kw in (dict(next_tokens=tokens[:2]), dict(accepted=tokens[4:]), dict(next_tokens=cu[1:]), dict(accepted=buf[:2], next_tokens=buf[1:3])):
        with pytest.raises(_lib.MGError):
            K().verify_drafts(logits, tokens, cu, u, **kw)
    K().verify_drafts(logits, tokens, cu, u, accepted=buf[:2], next_tokens=buf[2:4])  # side by side is well
    want = verify_oracle(logits, tokens.cpu().numpy(), cu.cpu().numpy(), u.cpu().numpy(), None, None)
    assert buf.tolist() == want[0] + want[1] + [0] and errors()[0] == 0


@pytest.mark.parametrize("probs", [False, True])
@pytest.mark.parametrize("t", [1e-44, 1e-40, 4e-39, 1e-37, 1e-30, 1e30])
def test_verify_extreme_temperatures(t, probs):
    """Any T > 0 is a temperature, the smallest numbers that fp32 has among them, where the softmax is the maximum's alone; and
    large ones, where all tokens are nearly alike."""
    logits, tokens, cu, u, q = verify_case([3, 0, 2, 5], 20000, probs, 8)
    temps = np.full(4, t, np.float32)
    got = K().verify_drafts(logits, i32(tokens), i32(cu), u, draft_probs=q, temperatures=torch.from_numpy(temps).cuda())
    want = verify_oracle(logits, tokens, cu, u.cpu().numpy(), q, temps)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    assert errors()[0] == 0


def test_verify_greedy_takes_nan_as_the_maximum():
    logits, tokens, cu, u, _ = verify_case([1], 300, False, 4)
    logits[0, 77] = math.nan
    tokens = tokens.copy()
    tokens[1] = 77
    acc, nxt = K().verify_drafts(logits, i32(tokens), i32(cu), u, temperatures=torch.zeros(1, device="cuda"))
    assert acc.item() == 1 and nxt.item() == int(logits[1].argmax())
    assert errors()[0] == 0
