"""The ragged path through the backend and the engine on the GPU: prompts of different lengths in one batch, padded
batches, passes that cut prompts, speculative verification, per-head norms, the scheduler's packed prefill. Each is
held to the same backend's request-by-request path (the bf16 tolerance of the other model tests: the two group the same
arithmetic into different launches) or to the 64-bit oracle model."""

import numpy as np
import pytest
import torch

from oracle import model as omodel
from tests._hf_models import TINY, make_hf_model, prompt_ids

pytestmark = pytest.mark.gpu

ATOL, RTOL = 1e-2, 2e-2


def close(got, want, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    err = np.abs(got - want)
    bad = err > ATOL + RTOL * np.abs(want)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} outside tolerance, max err {err.max():.3e}"


def backend(model=None, **kw):
    from microgen_b200.backends import B200QuantizedBackend
    be = B200QuantizedBackend(**{**dict(max_batch=4, max_seq_len=256, free_list_seed=5), **kw})
    if model is not None:
        be.load_model("tiny", model_instance=model)
    return be


def prompts_of(V, lens, seed=0):
    return [prompt_ids(V, n, seed=seed + i) for i, n in enumerate(lens)]


def one_by_one(be, prompts):
    """Logits after each prompt and the caches, each prompt in a batch of its own."""
    out = [be.prefill(torch.tensor([p])) for p in prompts]
    return np.concatenate([lg.float().cpu().numpy() for lg, _ in out]), [c for _, c in out]


def kv_rows(be, table):
    eng = be.engine
    pos = range(table.num_tokens)
    at = lambda pool: torch.stack([pool[:, table.physical_blocks[p // 16].block_id, :, p % 16].float() for p in pos])
    k, v = at(eng.pool.k), at(eng.pool.v)
    if eng.pool.quantize:
        sc = lambda s: torch.stack([s[:, table.physical_blocks[p // 16].block_id, :, p % 16] for p in pos])
        k, v = k * sc(eng.pool.k_scale)[..., None], v * sc(eng.pool.v_scale)[..., None]
    return torch.stack([k, v]).cpu().numpy()


@pytest.mark.parametrize("family", ["llama", "qwen2", "gpt2"])
@pytest.mark.parametrize("kv8", [False, True])
def test_ragged_prefill_and_decode(family, kv8):
    shape = TINY[family]
    model, _ = make_hf_model(shape, seed=0)
    be, ref = backend(model, quantize_kv=kv8), backend(model, quantize_kv=kv8)
    prompts = prompts_of(shape["vocab"], [1, 37, 130, 16], seed=3)
    lg, cache = be.prefill_ragged(prompts)
    want, caches = one_by_one(ref, prompts)
    close(lg.cpu().numpy(), want, "prompt logits")
    # (int8 codes of the two paths may differ by a step where a value lies between two)
    for t, c in zip(cache.tables, caches):
        a, b = kv_rows(be, t), kv_rows(ref, c.tables[0])
        if kv8:
            assert np.abs(a - b).max() <= np.abs(b).max() / 127 * 1.01 + ATOL
        else:
            close(a, b, "K/V")
    assert be.sample(lg)[:, 0].tolist() == lg.argmax(-1).tolist()  # the device's greedy tokens are these logits'
    for step in range(3):
        tok = torch.tensor([[int(want[i].argmax())] for i in range(4)])
        lg, cache = be.decode(tok, cache=cache)
        want = np.concatenate([ref.decode(tok[i:i + 1], cache=c)[0].cpu().numpy() for i, c in enumerate(caches)])
        close(lg.cpu().numpy(), want, f"decode step {step}")


def test_padded_batch_equals_its_prompts():
    shape = TINY["llama"]
    model, _ = make_hf_model(shape, seed=1)
    be, ref = backend(model), backend(model)
    lens = [5, 33, 20]
    prompts = prompts_of(shape["vocab"], lens, seed=9)
    want, _ = one_by_one(ref, prompts)
    ids = torch.zeros((3, 33), dtype=torch.long)
    mask = torch.zeros_like(ids)
    for i, p in enumerate(prompts):
        at = 33 - len(p) if i != 2 else 0  # the last one is padded behind
        ids[i, at:at + len(p)] = torch.tensor(p)
        mask[i, at:at + len(p)] = 1
    lg, cache = be.prefill(ids, attention_mask=mask)
    close(lg.cpu().numpy(), want, "padded logits")
    assert [t.num_tokens for t in cache.tables] == lens
    cache.free()
    assert be.allocator.get_num_allocated_blocks() == 0


def test_passes_cut_prompts_and_caches_continue():
    """A row budget smaller than the prompts, and a second call that continues the first's cache."""
    shape = TINY["qwen2"]
    model, _ = make_hf_model(shape, seed=2)
    be, ref = backend(model), backend(model)
    be.engine.RAGGED_ROWS = 24
    prompts = prompts_of(shape["vocab"], [70, 3, 41], seed=20)
    lg, cache = be.prefill_ragged(prompts)
    want, _ = one_by_one(ref, prompts)
    close(lg.cpu().numpy(), want, "cut prompts")
    more = prompts_of(shape["vocab"], [2, 50, 1], seed=50)
    lg, cache = be.prefill_ragged(more, cache=cache)
    want, _ = one_by_one(ref, [a + b for a, b in zip(prompts, more)])
    close(lg.cpu().numpy(), want, "continued")
    every = be.engine.forward_ragged([p[-30:] for p in (prompts[0], prompts[2])], [40, 11],
                                     np.stack([np.pad(t.block_ids(), (0, 16 - t.num_blocks())) for t in
                                               (cache.tables[0], cache.tables[2])]), all_logits=True)
    assert every.shape == (60, shape["vocab"])  # (cut into three passes; rows in the requests' order)


@pytest.mark.parametrize("family,kv8", [("llama", False), ("gpt2", True)])
def test_greedy_verification_gives_the_greedy_stream(family, kv8):
    """Drafts right, wrong from some place on, and missing: with temperature 0 the accepted tokens are the model's own
    greedy stream, and the cache afterwards is the one that decoding it would leave."""
    shape = TINY[family]
    model, _ = make_hf_model(shape, seed=3)
    V = shape["vocab"]
    be, ref = backend(model, quantize_kv=kv8), backend(model, quantize_kv=kv8)
    prompts = prompts_of(V, [12, 31, 47], seed=7)
    lg, cache = be.prefill_ragged(prompts)
    tok = be.sample(lg)
    streams = []
    for p in prompts:
        l, c = ref.prefill(torch.tensor([p]))
        s = []
        for _ in range(16):
            s.append(int(l.argmax()))
            l, c = ref.decode(torch.tensor([[s[-1]]]), cache=c)
        streams.append(s)
    out = [[int(t)] for t in tok[:, 0]]
    for k, wrong in ((4, None), (3, 1), (0, None), (5, 0)):
        drafts = []
        for i, s in enumerate(streams):
            d = list(s[len(out[i]):len(out[i]) + k])
            if i == 1 and wrong is not None and len(d) > wrong:
                d[wrong] = (d[wrong] + 1) % V
            drafts.append(d if i != 2 else d[:1])
        new, cache = be.verify(torch.tensor([o[-1] for o in out]), drafts, cache, temperatures=0.0)
        for i, n in enumerate(new):
            out[i] += n
            assert 1 <= len(n) <= len(drafts[i]) + 1
            assert cache.tables[i].num_tokens == len(prompts[i]) + len(out[i]) - 1
    for p, o in zip(prompts, out):  # teacher-forced: every token is the best one, or within the tolerance of it
        l, c = ref.prefill(torch.tensor([p]))
        for t in o:
            row = l.float()[0]
            assert float(row.max() - row[t]) <= 2 * (ATOL + RTOL * float(row.abs().max()))
            l, c = ref.decode(torch.tensor([[t]]), cache=c)
    assert sum(len(o) for o in out) > 3 * 5  # four steps give five tokens without a draft: right drafts were accepted
    cache.free()
    assert be.allocator.get_num_allocated_blocks() == 0


def test_sampled_verification_follows_the_rule():
    """With probabilities and given uniform numbers: the same answer as the rule applied to the pass's own logits."""
    from tests.test_gpu_ragged import verify_oracle
    shape = TINY["llama"]
    model, _ = make_hf_model(shape, seed=4)
    V = shape["vocab"]
    be = backend(model)
    prompts = prompts_of(V, [9, 20], seed=70)
    _, cache = be.prefill_ragged(prompts)
    g = torch.Generator().manual_seed(5)
    drafts = [[3, 9, 100], [44]]
    probs = [torch.softmax(torch.randn(len(d), V, generator=g) * 0.3, -1) for d in drafts]
    u = torch.rand(6, generator=g)
    lens = [t.num_tokens for t in cache.tables]
    before = be._grow(cache.tables, [4, 2])
    logits = be.engine.forward_ragged([[1] + drafts[0], [2] + drafts[1]], before, cache.mirror.update(cache.tables), all_logits=True)
    be._shrink(cache.tables, before)
    flat = [1] + drafts[0] + [2] + drafts[1]
    q = torch.zeros(6, V)
    q[0:3], q[4:5] = probs[0], probs[1]
    acc, nxt = verify_oracle(logits, flat, [0, 4, 6], u.numpy(), q, np.array([0.7, 1.0], np.float32))
    got, cache = be.verify([1, 2], drafts, cache, draft_probs=probs, temperatures=[0.7, 1.0], uniforms=u)
    assert got == [d[:a] + [t] for d, a, t in zip(drafts, acc, nxt)]
    assert [t.num_tokens for t in cache.tables] == [n + 1 + a for n, a in zip(lens, acc)]


def test_verify_takes_strided_numbers_of_either_device():
    shape = TINY["llama"]
    model, _ = make_hf_model(shape, seed=4)
    be = backend(model)
    _, cache = be.prefill_ragged(prompts_of(shape["vocab"], [9, 20], seed=70))
    start = [t.num_tokens for t in cache.tables]
    u, temps = torch.rand((5, 3), generator=torch.Generator().manual_seed(2)), torch.tensor([[0.7, 9.0], [1.0, 9.0]])
    answers = []
    for dev in ("cpu", "cuda"):
        for strided in (False, True):
            uu, tt = (x.to(dev)[:, 0] for x in (u, temps))
            if not strided:
                uu, tt = uu.contiguous(), tt.contiguous()
            got, cache = be.verify([1, 2], [[3, 9], [44]], cache, temperatures=tt, uniforms=uu)
            answers.append(got)
            be._shrink(cache.tables, start)
    assert all(a == answers[0] for a in answers)


def test_verify_failure_leaves_the_cache_as_it_was():
    shape = TINY["llama"]
    model, _ = make_hf_model(shape, seed=4)
    be = backend(model, num_blocks=3)
    _, cache = be.prefill_ragged([prompt_ids(shape["vocab"], 30, seed=1)])
    with pytest.raises(MemoryError):
        be.verify([1], [[2] * 20], cache)
    with pytest.raises(ValueError):
        be.verify([1], [[2]], cache, draft_probs=[torch.zeros(2, 5)])
    assert cache.tables[0].num_tokens == 30 and cache.tables[0].num_blocks() == 2
    got, cache = be.verify([1], [[2, 3]], cache, temperatures=0.0)
    assert cache.tables[0].num_tokens == 30 + len(got[0])


@pytest.mark.parametrize("chunk", [0, 64])
def test_per_head_norms_against_the_oracle(chunk):
    """A checkpoint with q_norm / k_norm weights: prefill (stepwise, chunked and packed) and decode against the oracle."""
    from microgen_b200.model_spec import spec_from_hf_config
    model, state = make_hf_model(TINY["llama"], seed=6)
    rng = np.random.default_rng(0)
    state = dict(state)
    for i in range(2):
        for n in "qk":
            state[f"model.layers.{i}.self_attn.{n}_norm.weight"] = (1 + 0.5 * rng.standard_normal(32)).astype(np.float32)
    sp = spec_from_hf_config(model.config)
    om = omodel.OracleModel(omodel.Spec(**{k: getattr(sp, k) for k in omodel.Spec.__dataclass_fields__}), state)
    be = backend(prefill_chunk=chunk)
    be.load_state(sp, {k: torch.from_numpy(np.asarray(v)) for k, v in state.items()})
    prompts = prompts_of(512, [19, 19], seed=30)
    want = []
    for p in prompts:
        c = om.new_cache()
        for t, tk in enumerate(p):
            lg = om.step(tk, t, c)
        want.append((lg, om.step(7, len(p), c)))
    lg, cache = be.prefill(torch.tensor(prompts))
    close(lg.cpu().numpy(), [w[0] for w in want], "prefill")
    lg, _ = be.decode(torch.tensor([[7], [7]]), cache=cache)
    close(lg.cpu().numpy(), [w[1] for w in want], "decode")
    lg, cache = be.prefill_ragged(prompts)
    close(lg.cpu().numpy(), [w[0] for w in want], "packed")
    plain = omodel.OracleModel(om.spec, {k: v for k, v in state.items() if "_norm.weight" not in k or "self_attn" not in k})
    c = plain.new_cache()
    for t, tk in enumerate(prompts[0]):
        without = plain.step(tk, t, c)
    assert np.abs(without - want[0][0]).max() > 10 * ATOL  # the norms matter in this case


def test_scheduler_with_packed_prefill():
    from microgen_b200.scheduler import BatchedScheduler, Request, RequestStatus
    shape = TINY["llama"]
    model, _ = make_hf_model(shape, seed=0)
    be = backend(model)
    reqs = [Request(request_id=f"r{i}", prompt="", prompt_ids=prompt_ids(shape["vocab"], n, seed=60 + n), max_new_tokens=5,
                    temperature=0.0) for i, n in enumerate((3, 50, 17, 29, 9))]
    sch = BatchedScheduler(be, max_batch_size=4, packed_prefill=True)
    for r in reqs:
        sch.add_request(r)
    sch.run_until_complete()
    ref = backend(model)
    for r in reqs:
        assert r.status == RequestStatus.COMPLETED and len(r.generated_token_ids) == 5
        lg, c = ref.prefill(torch.tensor([r.prompt_ids]))
        for t in r.generated_token_ids:  # teacher-forced: the chosen token is the best one, or within the tolerance of it
            row = lg.float()[0]
            assert float(row.max() - row[t]) <= 2 * (ATOL + RTOL * float(row.abs().max()))
            lg, c = ref.decode(torch.tensor([[t]]), cache=c)
    assert be.allocator.get_num_allocated_blocks() == 0
