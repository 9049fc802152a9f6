"""8-bit integer experts without a GPU: the header and its exports, the oracle, and the refusals
of the C ABI and the wrappers."""

import re
from types import SimpleNamespace

import pytest
import torch

import bench_profiles
from nanotitan_amd import build, capi, moe_ops
from nanotitan_amd.layer import Int8ExpertFFN, MoE
from nanotitan_amd.moe_ops import Int8Weight
from tests import int8_oracle as O
from tests.conftest import ROOT

F32, F64, F16, BF = capi.NT_F32, capi.NT_F64, capi.NT_F16, capi.NT_BF16
P = 4096  # a non-null, aligned address: none of these calls gets as far as using it


def test_exports_are_what_the_header_declares():
    text = (ROOT / "include" / "nanotitan_int8.h").read_text()
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"\b(nt_[a-z_0-9]+)\s*\(", text))
    assert names == set(capi.INT8_EXPORTS)
    assert not names & set(capi.EXPORTS)
    lib = capi.load()
    assert all(hasattr(lib, n) for n in names)


def test_sources_are_beside_the_profiled_ones():
    assert not set(build.INT8_SOURCES) & (set(build.HIP_SOURCES)
                                          | set(bench_profiles.PROFILED_SOURCES))
    for name in build.INT8_SOURCES:
        assert (build.CSRC / name).is_file()


def test_oracle():
    q, s = O.held(torch.tensor([[127.0, 0.5, 1.5, -2.5, -127.0], [0.0] * 5,
                                [1.0, 0.5, float("nan"), 0.0, 0.0]]), 1)
    assert q.tolist() == [[127, 0, 2, -2, -127], [0] * 5, [0] * 5]
    assert s[:2, 0].tolist() == [1.0, 2.0**-126] and bool(s[2].isnan())
    w = torch.arange(2 * 70 * 130).view(2, 70, 130) % 251 - 125
    b = O.blocks(w)
    assert b.shape == (2, 3, 2, 4, 4, 16, 16)
    # k = 69 = 64 + 5, n = 129 = 128 + 1: t 0, i 1, g 0, byte 5
    assert int(b[1, 2, 1, 0, 0, 1, 5]) == int(w[1, 69, 129])
    # k = 37: g 2, byte 5; n = 64 + 43: 43 = 32 + 8 + 3: t 2, i 11
    assert int(b[0, 1, 0, 2, 2, 11, 5]) == int(w[0, 37, 107])
    assert int((b != 0).sum()) == int((w != 0).sum())


def test_sizes():
    lib = capi.load()
    assert [lib.nt_int8_pitch(f) for f in (1, 127, 128, 129, 14336)] == [128, 128, 128, 256, 14336]
    assert lib.nt_int8_rows_bytes(17, 129) == 32 * 256 and lib.nt_int8_rows_bytes(0, 5) == 0
    assert lib.nt_int8_rows_bytes(-1, 5) == 0
    assert lib.nt_int8_weight_bytes(3, 129, 65) == 3 * 256 * 128
    assert lib.nt_int8_weight_bytes(0, 128, 64) == 0
    assert lib.nt_int8_weight_bytes(1025, 128, 64) == 0
    assert lib.nt_int8_weight_bytes(1, capi.NT_INT8_MAX_K + 1, 64) == 0
    assert lib.nt_int8_weight_workspace_bytes(3, 65) == 3 * 65 * 4


MAX_K = capi.NT_INT8_MAX_K


@pytest.mark.parametrize("fn,args,code", [
    ("nt_int8_rows", (F64, P, 4, 8, P, P, None), capi.NT_ERR_DTYPE),
    ("nt_int8_rows", (BF, P, -1, 8, P, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows", (BF, P, 4, 0, P, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows", (BF, None, 4, 8, P, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows", (BF, P, 4, 8, P + 8, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows", (BF, P, 4, 8, P, None, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows", (BF, P, 4, MAX_K + 1, P, P, None), capi.NT_ERR_TOO_LARGE),
    ("nt_int8_rows", (BF, P, 2**24, 8, P, P, None), capi.NT_ERR_TOO_LARGE),
    ("nt_int8_rows", (BF, None, 0, 8, None, None, None), capi.NT_OK),
    ("nt_int8_rows_decode", (9, P, P, 4, 8, P, None), capi.NT_ERR_DTYPE),
    ("nt_int8_rows_decode", (BF, P, P, 4, 8, None, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows_decode", (BF, P + 4, P, 4, 8, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_rows_decode", (BF, None, None, 0, 8, None, None), capi.NT_OK),
    ("nt_int8_weight", (F64, P, 1, 8, 8, P, P, P, 32, None), capi.NT_ERR_DTYPE),
    ("nt_int8_weight", (BF, P, 0, 8, 8, P, P, P, 32, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_weight", (BF, P, 1025, 8, 8, P, P, P, 2**20, None), capi.NT_ERR_TOO_MANY_EXPERTS),
    ("nt_int8_weight", (BF, P, 1, MAX_K + 1, 8, P, P, P, 32, None), capi.NT_ERR_TOO_LARGE),
    ("nt_int8_weight", (BF, P, 1, 8, 2**22 + 1, P, P, P, 2**30, None), capi.NT_ERR_TOO_LARGE),
    ("nt_int8_weight", (BF, P, 1, 8, 8, P + 1, P, P, 32, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_weight", (BF, P, 1, 8, 8, P, P, P, 31, None), capi.NT_ERR_WORKSPACE),
    ("nt_int8_weight", (BF, P, 1, 8, 8, P, P, None, 32, None), capi.NT_ERR_WORKSPACE),
    ("nt_int8_weight", (BF, P, 1, 8, 8, P, P, P + 2, 32, None), capi.NT_ERR_WORKSPACE),
    ("nt_int8_weight_decode", (BF, P, None, 1, 8, 8, P, None), capi.NT_ERR_INVALID_ARG),
    ("nt_int8_weight_decode", (7, P, P, 1, 8, 8, P, None), capi.NT_ERR_DTYPE)])
def test_rows_and_weights_refuse(fn, args, code):
    assert getattr(capi.load(), fn)(*args) == code


def _gemm(**over):
    a = dict(dtype=BF, x=P, xs=P, offsets=P, w=P, ws=P, E=2, A=4, K=8, N=8, out=P)
    a.update(over)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(dtype=F64), capi.NT_ERR_DTYPE), (dict(E=0), capi.NT_ERR_INVALID_ARG),
    (dict(A=-1), capi.NT_ERR_INVALID_ARG), (dict(K=0), capi.NT_ERR_INVALID_ARG),
    (dict(N=0), capi.NT_ERR_INVALID_ARG), (dict(E=1025), capi.NT_ERR_TOO_MANY_EXPERTS),
    (dict(K=MAX_K + 1), capi.NT_ERR_TOO_LARGE), (dict(N=2**22 + 1), capi.NT_ERR_TOO_LARGE),
    (dict(A=2**24), capi.NT_ERR_TOO_LARGE), (dict(offsets=None), capi.NT_ERR_INVALID_ARG),
    (dict(x=None), capi.NT_ERR_INVALID_ARG), (dict(x=P + 8), capi.NT_ERR_INVALID_ARG),
    (dict(xs=None), capi.NT_ERR_INVALID_ARG), (dict(w=None), capi.NT_ERR_INVALID_ARG),
    (dict(w=P + 1), capi.NT_ERR_INVALID_ARG), (dict(ws=None), capi.NT_ERR_INVALID_ARG),
    (dict(out=None), capi.NT_ERR_INVALID_ARG), (dict(A=0, x=None, out=None), capi.NT_OK)])
def test_products_refuse(over, code):
    lib, a = capi.load(), _gemm(**over)
    ins = [a[n] for n in ("dtype", "x", "xs", "offsets", "w", "ws")]
    sizes = [a[n] for n in ("E", "A", "K", "N")]
    assert lib.nt_int8_grouped_gemm(*ins, *sizes, a["out"], None) == code
    assert lib.nt_int8_grouped_gemm_gelu(*ins, *sizes, a["out"], None, None) == code
    assert lib.nt_int8_grouped_gemm_swiglu(*ins, P, P, *sizes, a["out"], None, None, None) == code


@pytest.mark.parametrize("over,code", [
    (dict(dtype=F64), capi.NT_ERR_DTYPE), (dict(E=0), capi.NT_ERR_INVALID_ARG),
    (dict(K=0), capi.NT_ERR_INVALID_ARG), (dict(offsets=None), capi.NT_ERR_INVALID_ARG),
    (dict(x=None), capi.NT_ERR_INVALID_ARG), (dict(w=None), capi.NT_ERR_INVALID_ARG),
    (dict(out=None), capi.NT_ERR_INVALID_ARG), (dict(A=2**24), capi.NT_ERR_TOO_LARGE),
    (dict(ws_bytes=100), capi.NT_ERR_WORKSPACE), (dict(ws=None), capi.NT_ERR_WORKSPACE),
    (dict(ws=P + 8), capi.NT_ERR_WORKSPACE), (dict(A=0, x=None, out=None, ws=None), capi.NT_OK)])
def test_linear_refuses(over, code):
    lib, a = capi.load(), dict(dtype=BF, x=P, offsets=P, w=P, s=P, E=2, A=4, K=8, N=8, out=P, ws=P,
                               ws_bytes=2**20)
    a.update(over)
    head = [a[n] for n in ("dtype", "x", "offsets", "w", "s")]
    sizes = [a[n] for n in ("E", "A", "K", "N")]
    tail = [a["ws"], a["ws_bytes"], None]
    assert lib.nt_int8_linear(*head, *sizes, a["out"], *tail) == code
    assert lib.nt_int8_linear_gelu(*head, *sizes, a["out"], None, *tail) == code
    assert lib.nt_int8_linear_swiglu(*head, P, P, *sizes, a["out"], None, None, *tail) == code
    assert lib.nt_int8_linear_workspace_bytes(17, 129) == 32 * 256 + 80


def test_swiglu_refuses_half_of_a_pair():
    a = _gemm()
    ins = [a[n] for n in ("dtype", "x", "xs", "offsets", "w", "ws")]
    fn = capi.load().nt_int8_grouped_gemm_swiglu
    for w2, s2, gate, value in ((None, P, None, None), (P, None, None, None), (P, P, P, None),
                                (P, P, None, P), (P + 8, P, None, None)):
        assert fn(*ins, w2, s2, 2, 4, 8, 8, P, gate, value, None) == capi.NT_ERR_INVALID_ARG


def _grad(**over):
    a = dict(dtype=BF, w=P, s=P, offsets=P, dout=P, pitch=16, E=2, A=4, K=9, N=16, out=P)
    a.update(over)
    return a


@pytest.mark.parametrize("over,code", [
    (dict(dtype=9), capi.NT_ERR_DTYPE), (dict(E=0), capi.NT_ERR_INVALID_ARG),
    (dict(A=-1), capi.NT_ERR_INVALID_ARG), (dict(K=0), capi.NT_ERR_INVALID_ARG),
    (dict(E=1025), capi.NT_ERR_TOO_MANY_EXPERTS),
    (dict(K=MAX_K + 1), capi.NT_ERR_TOO_LARGE), (dict(N=2**22 + 8), capi.NT_ERR_TOO_LARGE),
    (dict(A=2**24), capi.NT_ERR_TOO_LARGE), (dict(offsets=None), capi.NT_ERR_INVALID_ARG),
    (dict(w=None), capi.NT_ERR_INVALID_ARG), (dict(w=P + 8), capi.NT_ERR_INVALID_ARG),
    (dict(dout=None), capi.NT_ERR_INVALID_ARG),
    (dict(dout=P + 2), capi.NT_ERR_INVALID_ARG), (dict(out=None), capi.NT_ERR_INVALID_ARG),
    (dict(A=0, dout=None, out=None), capi.NT_OK)])
def test_gradients_refuse(over, code):
    lib, a = capi.load(), _grad(**over)
    head = [a[n] for n in ("dtype", "w", "s", "offsets", "dout", "pitch")]
    sizes = [a[n] for n in ("E", "A", "K", "N")]
    assert lib.nt_int8_grouped_gemm_dx(*head, *sizes, a["out"], None) == code
    assert lib.nt_int8_grouped_gemm_dx_gelu(*head, P, P, *sizes, a["out"], None) == code
    assert lib.nt_int8_grouped_gemm_dx_swiglu(*head, P, P, P, P, *sizes, a["out"], P, None) == code
    assert lib.nt_int8_grouped_gemm_dx_terms(a["dtype"], a["w"], None, a["offsets"], a["dout"],
                                             None, *sizes, a["out"], None) == code


def test_gradients_refuse_missing_inputs():
    lib = capi.load()
    sizes, bad = [2, 4, 9, 16], capi.NT_ERR_INVALID_ARG
    head = [BF, P, P, P, P, 16]
    for pitch in (8, 20):  # below N, and no multiple of 8
        assert lib.nt_int8_grouped_gemm_dx(*head[:5], pitch, *sizes, P, None) == bad
    assert lib.nt_int8_grouped_gemm_dx(*head[:5], 2**22 + 8, *sizes, P,
                                       None) == capi.NT_ERR_TOO_LARGE
    assert lib.nt_int8_grouped_gemm_dx(BF, P, None, *head[3:], *sizes, P, None) == bad
    for i in range(2):
        args = [None if i == j else P for j in range(2)]
        assert lib.nt_int8_grouped_gemm_dx_gelu(*head, *args, *sizes, P, None) == bad
    assert lib.nt_int8_grouped_gemm_dx_gelu(*head, P, P, *sizes, P + 8, None) == bad
    for i in range(4):
        args = [None if i == j else P for j in range(4)]
        assert lib.nt_int8_grouped_gemm_dx_swiglu(*head, *args, *sizes, P, P, None) == bad
    assert lib.nt_int8_grouped_gemm_dx_swiglu(*head, P, P, P, P, *sizes, P, None, None) == bad
    assert lib.nt_int8_grouped_gemm_dx_swiglu(*head, P, P, P, P, *sizes, P, P + 8, None) == bad
    for two in ((P, None), (None, P), (P, P + 8), (P + 8, P)):
        assert lib.nt_int8_grouped_gemm_dx_terms(BF, P, two[0], P, P, two[1], *sizes, P,
                                                 None) == bad


def test_terms():
    lib = capi.load()
    size = lib.nt_int8_terms_bytes
    assert size(BF, 5, 129) == 2 * 5 * 256 * 2 and size(F32, 5, 129) == 3 * 5 * 256 * 2
    assert size(BF, 0, 4) == size(BF, 4, 0) == size(9, 4, 4) == 0
    assert size(BF, 4, 2**22 + 1) == size(BF, 2**24, 4) == 0
    good = [P, P, P, 2, 4, 9, P]
    for i, (v, code) in enumerate([(None, capi.NT_ERR_INVALID_ARG)] * 3 + [
            (0, capi.NT_ERR_INVALID_ARG), (2**24, capi.NT_ERR_TOO_LARGE),
            (0, capi.NT_ERR_INVALID_ARG), (P + 8, capi.NT_ERR_INVALID_ARG)]):
        assert lib.nt_int8_terms(*good[:i], v, *good[i + 1:], None) == code
    assert lib.nt_int8_terms(*good[:3], 1025, *good[4:], None) == capi.NT_ERR_TOO_MANY_EXPERTS
    assert lib.nt_int8_terms(None, None, None, 1, 0, 9, None, None) == capi.NT_OK


def _few(**over):
    a = dict(dtype=BF, x=P, router=P, logits=None, wu=P, su=P, wv=P, sv=P, wd=P, sd=P, T=4, E=8,
             k=2, d=64, f=128, gates=P, topk=P, out=P, ws=P, ws_bytes=2**30, stream=None)
    a.update(over)
    return list(a.values())


@pytest.mark.parametrize("over,code", [
    (dict(dtype=F64), capi.NT_ERR_DTYPE), (dict(T=65), capi.NT_ERR_TOO_LARGE),
    (dict(T=-1), capi.NT_ERR_INVALID_ARG), (dict(E=1025), capi.NT_ERR_TOO_MANY_EXPERTS),
    (dict(E=64, k=33), capi.NT_ERR_INVALID_ARG), (dict(k=9), capi.NT_ERR_INVALID_ARG),
    (dict(k=0), capi.NT_ERR_INVALID_ARG), (dict(d=0), capi.NT_ERR_INVALID_ARG),
    (dict(d=MAX_K + 1), capi.NT_ERR_TOO_LARGE), (dict(f=MAX_K + 1), capi.NT_ERR_TOO_LARGE),
    (dict(logits=P), capi.NT_ERR_INVALID_ARG), (dict(router=None), capi.NT_ERR_INVALID_ARG),
    (dict(sv=None), capi.NT_ERR_INVALID_ARG), (dict(wv=None), capi.NT_ERR_INVALID_ARG),
    (dict(wu=P + 8), capi.NT_ERR_INVALID_ARG), (dict(wd=P + 8), capi.NT_ERR_INVALID_ARG),
    (dict(sd=None), capi.NT_ERR_INVALID_ARG), (dict(out=None), capi.NT_ERR_INVALID_ARG),
    (dict(gates=None), capi.NT_ERR_INVALID_ARG), (dict(x=None), capi.NT_ERR_INVALID_ARG),
    (dict(ws=None), capi.NT_ERR_WORKSPACE), (dict(ws=P + 8), capi.NT_ERR_WORKSPACE),
    (dict(ws_bytes=64), capi.NT_ERR_WORKSPACE), (dict(T=0, x=None, ws=None), capi.NT_OK)])
def test_few_tokens_refuse(over, code):
    assert capi.load().nt_int8_moe_few_tokens(*_few(**over)) == code


def _weight(E, K, N):
    return Int8Weight(torch.zeros(E, -(-N // 64), O.pitch(K) // 64, 4, 4, 16, 16,
                                  dtype=torch.int8), torch.ones(E, N), (E, K, N))


def test_wrappers_refuse():
    x = torch.zeros(4, 64)
    w, down = _weight(2, 64, 96), _weight(2, 96, 64)
    for call in (lambda: moe_ops.int8_rows(x), lambda: moe_ops.int8_weight(torch.zeros(2, 8, 8)),
                 lambda: moe_ops.int8_grouped_gemm_fn(x, w, torch.zeros(3, dtype=torch.int32)),
                 lambda: moe_ops.int8_weight_decode(w, torch.float32),
                 lambda: moe_ops.int8_gelu_ffn_fn(x, w, down)):
        with pytest.raises(RuntimeError, match="must be a GPU tensor"):
            call()
    with pytest.raises(RuntimeError, match="expected an Int8Weight"):
        moe_ops.int8_grouped_gemm_fn(x, torch.zeros(2, 64, 96))
    with pytest.raises(RuntimeError, match="does not fit"):
        moe_ops.int8_grouped_gemm_fn(torch.zeros(4, 65), w)
    with pytest.raises(RuntimeError, match="do not fit"):
        moe_ops.int8_swiglu_ffn_fn(x, w, w, w)
    with pytest.raises(RuntimeError, match="do not fit"):
        moe_ops.int8_swiglu_ffn_fn(x, w, _weight(2, 64, 95), down)
    with pytest.raises(RuntimeError, match="with scales"):
        moe_ops.int8_grouped_gemm_fn(x, w._replace(shape=(2, 64, 97)))
    with pytest.raises(RuntimeError, match="all in 8 bits"):
        moe_ops.moe_few_tokens(x, (w, torch.zeros(2, 96, 64)), 1, logits=torch.zeros(4, 2))
    with pytest.raises(RuntimeError, match="no backward"):
        moe_ops.moe_few_tokens(x.requires_grad_(), (w, down), 1, logits=torch.zeros(4, 2))


def test_experts_of_others_are_refused():
    with pytest.raises(RuntimeError, match="Linear"):
        Int8ExpertFFN(torch.nn.Linear(4, 4))
    cfg = SimpleNamespace(num_experts=2, top_k=1, d_model=8, ffn_in=16, dtype=torch.float32,
                          moe_backend="hip", router_alpha=0.01)
    with pytest.raises(RuntimeError, match="must be a GPU tensor"):
        MoE(cfg).quantize_experts()
