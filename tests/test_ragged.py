"""Refusals of the ragged-batch operators that need no GPU: the C ABI's argument checks (before any CUDA call) and
the wrappers' checks of types, shapes and devices."""

import ctypes

import pytest
import torch

from microgen_b200 import _lib
from microgen_b200 import kernels as K

BAD, UNSUP = _lib.MG_ERR_INVALID_ARG, _lib.MG_ERR_UNSUPPORTED
P = ctypes.c_void_p(4096)  # an address that is only looked at


@pytest.fixture(scope="module")
def lib():
    from microgen_b200 import build
    build.build()
    return _lib.load()


def _plan(lib, b=2, rows=4, width=3, blocks=8, hq=8, hkv=2, d=64, q=P, work=P, nbytes=1 << 30):
    return lib.mg_ragged_plan(q, P, b, rows, P, width, blocks, None, None, 0, None, hq, hkv, d, P, P, P, P, P, P, P, work,
                              nbytes, None)


def test_plan_refusals(lib):
    n = ctypes.c_size_t(0)
    assert lib.mg_ragged_plan_bytes(64, 4, 24, 8, 128, ctypes.byref(n)) == 0 and n.value > 64
    assert lib.mg_ragged_plan_bytes(64, 4, 24, 7, 128, ctypes.byref(n)) == BAD       # heads that do not group
    assert lib.mg_ragged_plan_bytes(-1, 4, 24, 8, 128, ctypes.byref(n)) == BAD
    assert lib.mg_ragged_plan_bytes(64, 4, 24, 8, 128, None) == BAD
    assert lib.mg_ragged_plan_bytes(64, 4, 24, 8, 96, ctypes.byref(n)) == UNSUP      # head size
    assert lib.mg_ragged_plan_bytes(64, 4, 34, 2, 64, ctypes.byref(n)) == UNSUP      # 17 heads per K/V head
    assert lib.mg_ragged_plan_bytes(64, 8193, 24, 8, 128, ctypes.byref(n)) == UNSUP  # requests
    assert _plan(lib, b=-1) == BAD
    assert _plan(lib, width=0) == BAD
    assert _plan(lib, blocks=0) == BAD
    assert _plan(lib, q=None) == BAD
    assert _plan(lib, work=None) == BAD
    assert _plan(lib, work=ctypes.c_void_p(4104)) == BAD                              # alignment
    assert _plan(lib, nbytes=16) == BAD                                               # a work area too small
    assert _plan(lib, d=48) == UNSUP


def _append(lib, rows=3, ld=None, hq=8, hkv=2, d=64, qkv=P, ks=None, vs=None, cs=None, pos=None, max_pos=0, k=P):
    ld = (hq + 2 * hkv) * d if ld is None else ld
    return lib.mg_norm_rope_kv_append(qkv, 0, ld, rows, pos, cs, max_pos, P, None, None, 1e-6, hq, hkv, d, P, 1, k, P, ks,
                                      vs, 4, None)


def test_append_refusals(lib):
    assert _append(lib, rows=0) == 0                       # nothing to do, and no CUDA call
    assert _append(lib, rows=-1) == BAD
    assert _append(lib, hkv=3) == BAD
    assert _append(lib, ld=100) == BAD                     # rows that overlap
    assert _append(lib, ld=(8 + 4) * 64 + 2) == BAD        # row stride that breaks 16-byte loads
    assert _append(lib, qkv=ctypes.c_void_p(4100)) == BAD
    assert _append(lib, k=None) == BAD
    assert _append(lib, ks=P) == BAD                       # one of the two scale arrays
    assert _append(lib, cs=P, pos=None, max_pos=9) == BAD
    assert _append(lib, cs=P, pos=P, max_pos=0) == BAD
    assert _append(lib, d=80, ld=8000) == UNSUP


def _attn(lib, rows=4, hq=8, hkv=2, d=64, scale=0.1, q=P, ks=None, vs=None, nbytes=1 << 40, out=P, width=3):
    return lib.mg_ragged_attn(q, rows, P, P, ks, vs, 8, P, width, 2, 16, hq, hkv, d, ctypes.c_float(scale), P, out, P,
                              nbytes, None)


def test_attention_refusals(lib):
    assert _attn(lib, rows=0) == 0
    assert _attn(lib, rows=-1) == BAD
    assert _attn(lib, hkv=3) == BAD
    assert _attn(lib, scale=0.0) == BAD
    assert _attn(lib, scale=-0.1) == BAD
    assert _attn(lib, scale=float("nan")) == BAD
    assert _attn(lib, scale=float("inf")) == BAD
    assert _attn(lib, q=None) == BAD
    assert _attn(lib, q=ctypes.c_void_p(4104)) == BAD
    assert _attn(lib, out=None) == BAD
    assert _attn(lib, vs=P) == BAD
    assert _attn(lib, width=0) == BAD
    assert _attn(lib, nbytes=64) == BAD
    assert _attn(lib, d=256) == UNSUP
    assert _attn(lib, hq=34) == UNSUP


def test_outputs_over_their_inputs_are_refused(lib):
    n = 4 * 8 * 64 * 2  # bytes of the default q and out
    for out in (P, ctypes.c_void_p(P.value + n - 16), ctypes.c_void_p(P.value - n + 16)):
        assert _attn(lib, out=out) == BAD
    n = 3 * 8 * 64 * 2  # ... and of the default q_out, at P
    for qkv in (P, ctypes.c_void_p(P.value + n - 16), ctypes.c_void_p(P.value - 2048)):
        assert _append(lib, qkv=qkv) == BAD


def _verify(lib, rows=3, vocab=11, ld=11, ldq=11, b=2, logits=P, probs=None, ws=P, nbytes=1 << 20):
    return lib.mg_verify_drafts(logits, ld, rows, vocab, P, P, b, probs, ldq, P, None, P, P, ws, nbytes, None)


def test_verify_refusals(lib):
    assert _verify(lib, b=0, rows=0) == 0
    assert _verify(lib, rows=-1) == BAD
    assert _verify(lib, vocab=0) == BAD
    assert _verify(lib, ld=10) == BAD
    assert _verify(lib, probs=P, ldq=10) == BAD
    assert _verify(lib, logits=None) == BAD
    assert _verify(lib, ws=None) == BAD
    assert _verify(lib, nbytes=8) == BAD
    assert _verify(lib, rows=70000) == UNSUP
    assert _verify(lib, b=70000, nbytes=1 << 40) == UNSUP


def test_verify_outputs_over_inputs_are_refused(lib):
    """Requests are answered while others still read: no output may lie on an input, on the workspace or on the other output.
    (Only refusals are called here: the addresses are made up.)"""
    at = {n: 0x10000000 * (i + 1) for i, n in enumerate(("logits", "tokens", "cu", "probs", "u", "temps", "acc", "next", "ws"))}
    rows, vocab, b = 5, 100, 3

    def call(**kw):
        a = {k: ctypes.c_void_p(v) for k, v in {**at, **kw}.items()}
        return lib.mg_verify_drafts(a["logits"], vocab, rows, vocab, a["tokens"], a["cu"], b, a["probs"], vocab, a["u"], a["temps"],
                                    a["acc"], a["next"], a["ws"], 1 << 20, None)

    size = dict(logits=rows * vocab * 4, tokens=rows * 4, cu=(b + 1) * 4, probs=rows * vocab * 4, u=rows * 4, temps=b * 4, ws=512)
    for name, n in size.items():
        for out in ("acc", "next"):
            assert call(**{out: at[name]}) == BAD
            assert call(**{out: at[name] + n - 4}) == BAD
            assert call(**{out: at[name] - b * 4 + 4}) == BAD
    assert call(acc=at["next"]) == BAD and call(next=at["acc"] + 8) == BAD


def test_wrappers_refuse_host_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 12 * 64)
    pool = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        K.RaggedPlan(2, 8, 4, 8, 2, 64, "cpu")
    with pytest.raises(TypeError):
        K.norm_rope_kv_append(x, None, None, i, 8, 2, 64, pool, pool)
    with pytest.raises(ValueError):
        K.verify_drafts(torch.zeros(2, 5), i, torch.zeros(2, dtype=torch.int32), torch.zeros(2))
