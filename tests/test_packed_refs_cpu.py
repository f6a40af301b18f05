"""The packed-training operators' references against torch's autograd and against differences,
and what the entry points refuse, all without a device: arguments are checked before the runtime
is asked for."""
import ctypes
import math

import numpy as np
import pytest
import torch

import packed_ref as R
from vearo_amd import _abi as vh

r = np.random.default_rng(7)


def normal(*shape):
    return r.standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("causal", [True, False])
def test_attention_reference_is_autograds(causal):
    lens, Hq, Hk, D, scale = [3, 0, 1, 7], 4, 2, 5, 0.7
    q, k, v, do = normal(11, Hq, D), normal(11, Hk, D), normal(11, Hk, D), normal(11, Hq, D)
    val, tol = R.attention(q, k, v, do, lens, scale, causal)
    Q, K, V = (R.f64(x).requires_grad_() for x in (q, k, v))
    outs, t0 = [], 0
    for L in lens:
        s = slice(t0, t0 + L)
        t0 += L
        z = scale * torch.einsum("ihd,jhd->hij", Q[s], K[s].repeat_interleave(Hq // Hk, 1))
        if causal:
            z = z.masked_fill(torch.ones(L, L, dtype=torch.bool).triu(1), -math.inf)
        outs.append(torch.einsum("hij,jhd->ihd", torch.softmax(z, -1), V[s].repeat_interleave(Hq // Hk, 1)))
    o = torch.cat(outs)
    for n, x in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, (Q, K, V), R.f64(do)))):
        np.testing.assert_allclose(val[n], x.detach().numpy(), rtol=1e-12, atol=1e-13)
        # A wrong sign, a lost term or a neighbouring key is far beyond the bound.
        assert np.nanmax(tol[n]) < 1e-3


@pytest.mark.parametrize("interleaved", [0, 1])
def test_rope_reference_against_differences(interleaved):
    T, H, D, rot, eps, base = 3, 2, 6, 4, 1e-3, 100.0
    x, w, dy, pos = normal(T, H, D), 1 + 0.1 * normal(D), normal(T, H, D), np.array([0, 1, 1000.5], np.float32)
    val, _ = R.rope(x, w, dy, pos, eps, base, rot, interleaved)
    f = lambda a, b: (R.rope(a, b, dy, pos, eps, base, rot, interleaved)[0]["y"] * dy).sum()  # noqa: E731
    ux, uw, h = normal(T, H, D).astype(np.float64), normal(D).astype(np.float64), 1e-6
    num = (f(x + h * ux, w + h * uw) - f(x - h * ux, w - h * uw)) / (2 * h)
    assert abs(num - (val["dx"] * ux).sum() - (val["dw"] * uw).sum()) < 1e-7
    # A rotation keeps each pair's length; position 0 is none.
    np.testing.assert_allclose(val["y"][0], (R.f64(x[0]) / torch.sqrt((R.f64(x[0]) ** 2).mean(-1, keepdim=True) + eps)
                                             * R.f64(w)).numpy(), rtol=1e-12)


def test_linear_xent_reference_is_autograds():
    x, w = normal(9, 5), normal(13, 5)
    t = r.integers(0, 13, 9).astype(np.float32)
    t[[2, 5]] = -100
    val, tol = R.linear_xent(x, w, t, -100.0, 0.5)
    X, Y = R.f64(x).requires_grad_(), R.f64(w).requires_grad_()
    loss = torch.nn.functional.cross_entropy(X @ Y.T, torch.as_tensor(t).long(), ignore_index=-100)
    dx, dw = torch.autograd.grad(0.5 * loss, (X, Y))
    np.testing.assert_allclose(val["loss"][0], loss.item(), rtol=1e-13)
    np.testing.assert_allclose(val["dx"], dx.numpy(), rtol=1e-10, atol=1e-14)
    np.testing.assert_allclose(val["dw"], dw.numpy(), rtol=1e-10, atol=1e-14)
    none, _ = R.linear_xent(x, w, np.full(9, -100, np.float32), -100.0, 0.5)
    assert none["loss"][0] == 0 and not none["dx"].any() and not none["dw"].any()


# ----------------------------------------------------------------- refusals --
# Pointers are never followed here: an accepted call stops at the missing vh_init.
P = 4096


def refused(code, text, fn, *args):
    if vh._initialised:
        pytest.skip("runtime already initialised in this process")
    rc = getattr(vh.lib, fn)(*args)
    assert rc == code and text in vh.last_error(), (rc, vh.last_error())


def lay(*dims, strides=None):
    return ctypes.byref(vh.layout(dims, strides))


def rope_args(**kw):
    a = dict(q=P, ql=lay(4, 2, 8), k=P, kl=lay(4, 1, 8), wq=P, wk=P, pos=P, eps=1e-6, base=1e4, rot=8, inter=0, qo=P,
             qol=lay(4, 2, 8), ko=P, kol=lay(4, 1, 8), stream=None)
    return list((a | kw).values())


def rope_bwd_args(**kw):
    a = dict(q=P, ql=lay(4, 2, 8), k=P, kl=lay(4, 1, 8), wq=P, wk=P, pos=P, eps=1e-6, base=1e4, rot=8, inter=0, dqo=P,
             dqol=lay(4, 2, 8), dko=P, dkol=lay(4, 1, 8), dq=P, dql=lay(4, 2, 8), dk=P, dkl=lay(4, 1, 8), dwq=P, dwk=P,
             scratch=None, nb=0, stream=None)
    return list((a | kw).values())


@pytest.mark.parametrize("code,text,kw", [
    (vh.VH_ERR_NOT_INIT, "vh_init", {}),
    (vh.VH_ERR_INVALID, "rotary", {"rot": 10}), (vh.VH_ERR_INVALID, "rotary", {"rot": 3}),
    (vh.VH_ERR_INVALID, "rotary", {"rot": -2}), (vh.VH_ERR_INVALID, "eps", {"eps": -1.0}),
    (vh.VH_ERR_INVALID, "eps", {"eps": math.nan}), (vh.VH_ERR_INVALID, "base", {"base": 0.0}),
    (vh.VH_ERR_INVALID, "base", {"base": math.inf}), (vh.VH_ERR_INVALID, "null", {"q": None}),
    (vh.VH_ERR_INVALID, "null", {"pos": None}), (vh.VH_ERR_INVALID, "layout", {"ql": None}),
    (vh.VH_ERR_INVALID, "rank-3", {"ql": lay(4, 16)}), (vh.VH_ERR_INVALID, "shape", {"kl": lay(5, 1, 8)}),
    (vh.VH_ERR_UNSUPPORTED, "unit stride", {"ql": lay(4, 2, 8, strides=[16, 1, 2])}),
    (vh.VH_ERR_INVALID, "stride", {"ql": lay(4, 2, 8, strides=[-16, 8, 1])}),
])
def test_rope_refusals(code, text, kw):
    refused(code, text, "vh_qk_norm_rope_fwd", *rope_args(**kw))
    refused(code, text, "vh_qk_norm_rope_bwd", *rope_bwd_args(**kw))


@pytest.mark.parametrize("code,text,kw", [
    (vh.VH_ERR_INVALID, "null", {"qo": None}), (vh.VH_ERR_INVALID, "shape", {"qol": lay(4, 1, 8)}),
    (vh.VH_ERR_INVALID, "broadcast", {"qol": lay(4, 2, 8, strides=[16, 0, 1])}),
])
def test_rope_forward_refusals(code, text, kw):
    refused(code, text, "vh_qk_norm_rope_fwd", *rope_args(**kw))


@pytest.mark.parametrize("code,text,kw", [
    (vh.VH_ERR_INVALID, "null", {"dwq": None}), (vh.VH_ERR_INVALID, "null", {"dko": None}),
    (vh.VH_ERR_INVALID, "null", {"dk": None}), (vh.VH_ERR_INVALID, "shape", {"dqol": lay(4, 2, 6)}),
    (vh.VH_ERR_INVALID, "broadcast", {"dql": lay(4, 2, 8, strides=[0, 8, 1])}),
])
def test_rope_backward_refusals(code, text, kw):
    refused(code, text, "vh_qk_norm_rope_bwd", *rope_bwd_args(**kw))


def test_rope_head_size_limit():
    big = dict(ql=lay(4, 2, 258), kl=lay(4, 1, 258), qol=lay(4, 2, 258), kol=lay(4, 1, 258))
    refused(vh.VH_ERR_UNSUPPORTED, "head size", "vh_qk_norm_rope_fwd", *rope_args(**big))


def attention_args(**kw):
    a = dict(q=P, ql=lay(4, 4, 8), k=P, kl=lay(4, 2, 8), v=P, vl=lay(4, 2, 8), starts=P, n=2, scale=0.5, causal=1, o=P,
             ol=lay(4, 4, 8), lse=P, scratch=None, nb=0, stream=None)
    return list((a | kw).values())


def attention_bwd_args(**kw):
    a = dict(q=P, ql=lay(4, 4, 8), k=P, kl=lay(4, 2, 8), v=P, vl=lay(4, 2, 8), starts=P, n=2, scale=0.5, causal=1, o=P,
             ol=lay(4, 4, 8), lse=P, do=P, dol=lay(4, 4, 8), dq=P, dql=lay(4, 4, 8), dk=P, dkl=lay(4, 2, 8), dv=P,
             dvl=lay(4, 2, 8), scratch=None, nb=0, stream=None)
    return list((a | kw).values())


@pytest.mark.parametrize("code,text,kw", [
    (vh.VH_ERR_NOT_INIT, "vh_init", {}),
    (vh.VH_ERR_INVALID, "negative", {"n": -1}), (vh.VH_ERR_INVALID, "scale", {"scale": 0.0}),
    (vh.VH_ERR_INVALID, "scale", {"scale": -1.0}), (vh.VH_ERR_INVALID, "scale", {"scale": math.nan}),
    (vh.VH_ERR_INVALID, "scale", {"scale": math.inf}),
    (vh.VH_ERR_INVALID, "multiple", {"kl": lay(4, 3, 8), "vl": lay(4, 3, 8)}),
    (vh.VH_ERR_INVALID, "multiple", {"kl": lay(4, 0, 8), "vl": lay(4, 0, 8)}),
    (vh.VH_ERR_INVALID, "multiple", {"ql": lay(4, 0, 8), "ol": lay(4, 0, 8)}),
    (vh.VH_ERR_INVALID, "shape", {"vl": lay(4, 1, 8)}), (vh.VH_ERR_INVALID, "shape", {"ol": lay(4, 4, 6)}),
    (vh.VH_ERR_INVALID, "null", {"starts": None}), (vh.VH_ERR_INVALID, "null", {"lse": None}),
    (vh.VH_ERR_INVALID, "null", {"v": None}), (vh.VH_ERR_INVALID, "null", {"o": None}),
    (vh.VH_ERR_UNSUPPORTED, "unit stride", {"kl": lay(4, 2, 8, strides=[16, 1, 2])}),
    (vh.VH_ERR_UNSUPPORTED, "range", {"n": 2 ** 31}),
    (vh.VH_ERR_UNSUPPORTED, "range", {"ql": lay(2 ** 28 + 1, 4, 8), "ol": lay(2 ** 28 + 1, 4, 8),
                                      "kl": lay(2 ** 28 + 1, 2, 8), "vl": lay(2 ** 28 + 1, 2, 8)}),
])
def test_attention_refusals(code, text, kw):
    refused(code, text, "vh_packed_attention_fwd", *attention_args(**kw))
    refused(code, text, "vh_packed_attention_bwd", *attention_bwd_args(**kw))


@pytest.mark.parametrize("code,text,kw", [
    (vh.VH_ERR_INVALID, "null", {"do": None}), (vh.VH_ERR_INVALID, "null", {"dv": None}),
    (vh.VH_ERR_INVALID, "shape", {"dkl": lay(4, 4, 8)}), (vh.VH_ERR_INVALID, "shape", {"dol": lay(3, 4, 8)}),
    (vh.VH_ERR_INVALID, "broadcast", {"dvl": lay(4, 2, 8, strides=[16, 0, 1])}),
])
def test_attention_backward_refusals(code, text, kw):
    refused(code, text, "vh_packed_attention_bwd", *attention_bwd_args(**kw))


def test_attention_size_limits():
    big = {k: lay(4, h, 257) for k, h in (("ql", 4), ("kl", 2), ("vl", 2), ("ol", 4))}
    refused(vh.VH_ERR_UNSUPPORTED, "head size", "vh_packed_attention_fwd", *attention_args(**big))
    big = {k: lay(2 ** 31, h, 8) for k, h in (("ql", 4), ("kl", 2), ("vl", 2), ("ol", 4))}
    refused(vh.VH_ERR_UNSUPPORTED, "range", "vh_packed_attention_fwd", *attention_args(**big))


def xent_args(fn, **kw):
    a = dict(x=P, ldx=8, w=P, ldw=8, t=P, ignore=-100.0)
    a |= {"fwd": dict(loss=P, stats=P), "bwd": dict(stats=P, go=P, dx=P, lddx=8, dw=P, lddw=8),
          "fwd_bwd": dict(go=P, loss=P, dx=P, lddx=8, dw=P, lddw=8)}[fn]
    a |= dict(R=3, D=8, V=5, scratch=None, nb=0, stream=None)
    return list((a | {k: v for k, v in kw.items() if k in a}).values())


@pytest.mark.parametrize("fn", ["fwd", "bwd", "fwd_bwd"])
@pytest.mark.parametrize("code,text,kw", [
    (vh.VH_ERR_NOT_INIT, "vh_init", {}), (vh.VH_ERR_INVALID, "rows", {"R": 0}), (vh.VH_ERR_INVALID, "vocabulary", {"V": 0}),
    (vh.VH_ERR_INVALID, "width", {"D": 0}), (vh.VH_ERR_INVALID, "stride", {"ldx": 7}),
    (vh.VH_ERR_INVALID, "stride", {"ldw": 7}), (vh.VH_ERR_INVALID, "null", {"x": None}),
    (vh.VH_ERR_INVALID, "null", {"t": None}), (vh.VH_ERR_UNSUPPORTED, "int32", {"V": 2 ** 31}),
    (vh.VH_ERR_UNSUPPORTED, "int32", {"R": 2 ** 31}),
])
def test_linear_xent_refusals(fn, code, text, kw):
    refused(code, text, "vh_linear_cross_entropy_" + fn, *xent_args(fn, **kw))


@pytest.mark.parametrize("fn,text,kw", [
    ("fwd", "null", {"loss": None}), ("fwd", "null", {"stats": None}), ("fwd", "aligned", {"stats": P + 4}),
    ("bwd", "null", {"stats": None}), ("bwd", "null", {"go": None}), ("bwd", "stride", {"lddw": 7}),
    ("fwd_bwd", "null", {"dx": None}), ("fwd_bwd", "stride", {"lddx": 7}), ("fwd_bwd", "null", {"dw": None}),
])
def test_linear_xent_own_refusals(fn, text, kw):
    refused(vh.VH_ERR_INVALID, text, "vh_linear_cross_entropy_" + fn, *xent_args(fn, **kw))


def test_scratch_sizes():
    L = vh.lib
    assert L.vh_packed_attention_scratch_bytes(0, 1, 4, 2, 64, 1) == 0
    assert L.vh_packed_attention_scratch_bytes(16384, 8, 12, 4, 64, 1) >= 4 * 12 * 16384
    assert L.vh_qk_norm_rope_bwd_scratch_bytes(0, 64) == 0 < L.vh_qk_norm_rope_bwd_scratch_bytes(1, 1)
    assert L.vh_packed_attention_scratch_bytes(100, 1, 2, 4, 64, 1) > 0  # (head counts that a call refuses)
    # A gradient's pieces: three blocks of 683 MiB, and no less than 256 rows of logits. A forward: none.
    assert L.vh_linear_cross_entropy_scratch_bytes(65536, 768, 50257, 1) < 4 * 65536 * 50257 // 4
    assert L.vh_linear_cross_entropy_scratch_bytes(1024, 8, 4000000, 1) >= 4 * 256 * 4000000
    assert L.vh_linear_cross_entropy_scratch_bytes(65536, 768, 50257, 0) < 4 * 65536 * 50257 // 16
    assert L.vh_linear_cross_entropy_scratch_bytes(0, 8, 8, 1) == 0


def test_code_object_holds_every_kernel():
    import os

    from conftest import ROOT
    from test_abi_cpu import elf_symbols

    path = os.path.join(ROOT, "vearo_amd", "csrc", "_build", "packed_kernels.co")
    if not os.path.exists(path):
        pytest.skip("code object not built in-tree")
    names = {f"vh_rope_{d}_v{c}" for d in ("fwd", "bwd") for c in ("4_l4_n1", "4_l8_n1", "4_l16_n1", "4_l32_n1", "1_l64_n1",
                                                                  "1_l64_n2")}
    for dp in (32, 48, 64, 80, 96, 112, 128, 192, 256):
        names |= {f"vh_pa_{k}_{dp}" for k in ("prep", "fwd", "fold", "dq", "dkdv", "join")}
    names |= {f"vh_pa_bwd_{dp}" for dp in (32, 48, 64, 80, 96, 112, 128)}
    names |= {"vh_lx_" + k for k in ("count", "stats", "grad", "stats_grad", "loss", "split", "logits", "finish", "tops", "cols", "dz",
                                   "mm", "join")}
    assert not names - elf_symbols(path)
    assert open(path, "rb").read() in open(vh.LIB_PATH, "rb").read()
