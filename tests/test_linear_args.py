"""Refusals of the linear layers and of the routing calls: every argument check answers before
the device is touched, so it runs without a GPU; what passes them all fails on the null
stream (QGEMM_ERR_BAD_HANDLE)."""
import ctypes

import pytest

import qgemm
import qgemm._lib as L

A = 1 << 20  # an address that is never followed


def big(i):
    return (i + 1) << 32


LINEAR = dict(s=None, x=big(0), ldx=64, w=big(1), bias=0, residual=0, ldr=32, out=big(2),
              out_dtype=L.BF16, ldc=32, M=8, N=32, K=64, act=L.ACT_NONE, gated=0, algo=0)
W8A8 = dict(s=None, A=big(0), lda=64, B=big(1), sA=big(3), sB=big(4), bias=0, residual=0, ldr=32,
            out=big(2), out_dtype=L.BF16, ldc=32, M=8, N=32, K=64, act=L.ACT_NONE, gated=0, algo=0)
EXPERT = dict(s=None, x=big(0), ldx=64, w=big(1), bias=0, offsets=big(5), out=big(2),
              out_dtype=L.BF16, ldc=32, E=4, M=8, N=32, K=64, act=L.ACT_NONE, gated=0, algo=0)
W8A8_EXPERT = dict(s=None, A=big(0), lda=64, B=big(1), sA=big(3), sB=big(4), bias=0,
                   offsets=big(5), out=big(2), out_dtype=L.BF16, ldc=32, E=4, M=8, N=32, K=64,
                   act=L.ACT_NONE, gated=0, algo=0)
ROUTE = dict(s=None, logits=big(0), in_dtype=L.F32, weights=big(1), experts=big(2),
             offsets=big(3), rows=big(4), T=8, E=16, k=2, renormalize=1)
DISPATCH = dict(s=None, x=big(0), dtype=L.BF16, rows=big(1), out=big(2), T=8, k=2, K=64, R=16)
DISPATCH_Q = dict(s=None, x=big(0), in_dtype=L.BF16, rows=big(1), q=big(2), sA=big(3), T=8, k=2,
                  K=64, R=16)
COMBINE = dict(s=None, y=big(0), in_dtype=L.BF16, rows=big(1), weights=big(2), residual=0,
               out=big(3), out_dtype=L.BF16, T=8, k=2, N=64, R=16)
CALLS = {"qgemm_linear_bf16_nk": LINEAR, "qgemm_w8a8_linear": W8A8,
         "qgemm_expert_linear_bf16_nk": EXPERT, "qgemm_w8a8_expert_linear": W8A8_EXPERT,
         "qgemm_route_topk": ROUTE, "qgemm_dispatch_rows": DISPATCH,
         "qgemm_dispatch_rows_quantized": DISPATCH_Q, "qgemm_combine_rows": COMBINE}


def status(name, **change):
    args = dict(CALLS[name])
    assert set(change) <= set(args), change
    args.update(change)
    return L.try_call(name, *args.values())


@pytest.mark.parametrize("name", sorted(CALLS))
def test_good_arguments_fail_on_the_handle(name):
    assert status(name) == L.ERR_BAD_HANDLE


LINEARS = ["qgemm_linear_bf16_nk", "qgemm_w8a8_linear", "qgemm_expert_linear_bf16_nk",
           "qgemm_w8a8_expert_linear"]


@pytest.mark.parametrize("name", LINEARS)
def test_linear_refusals(name):
    i8 = "w8a8" in name
    x, ldx, w = ("A", "lda", "B") if i8 else ("x", "ldx", "w")
    bad = L.ERR_INVALID_ARG
    for change in ({"M": -1}, {"N": -1}, {"K": -1}, {"out_dtype": 2}, {"act": 5}, {"act": -1},
                   {"gated": 2}, {"algo": 3}, {ldx: 63}, {"ldc": 31}, {x: 0}, {w: 0}, {"out": 0},
                   {"out": big(0)}, {"out": big(0) + 64}, {"out": big(1)}):
        assert status(name, **change) == bad, change
    assert status(name, out=big(2) + 1) == L.ERR_BAD_ALIGN
    assert status(name, bias=big(6) + 2) == L.ERR_BAD_ALIGN
    assert status(name, out=big(2) + 2, out_dtype=L.F32) == L.ERR_BAD_ALIGN
    # nothing to do is no error, but for the handle; a gated layer is not one of no features
    assert status(name, M=0, **{x: 0}) == L.ERR_BAD_HANDLE
    assert status(name, N=0, out=0) == L.ERR_BAD_HANDLE
    # K = 0 leaves act(bias) + residual: the operands are not looked at
    assert status(name, K=0, **{x: 0, w: 0}) == L.ERR_BAD_HANDLE
    if i8:
        assert status(name, sA=0) == bad and status(name, sB=0) == bad
        assert status(name, K=131072, lda=131072) == L.ERR_UNSUPPORTED
    if "expert" in name:
        assert status(name, offsets=0) == bad
        assert status(name, E=0) == bad and status(name, E=1025) == bad
        assert status(name, E=1024, N=1 << 21, ldc=1 << 21) == L.ERR_UNSUPPORTED
    else:
        assert status(name, residual=big(7), ldr=31) == bad
        # the residual may be out itself, with its row pitch, and nothing in between
        assert status(name, residual=big(2)) == L.ERR_BAD_HANDLE
        assert status(name, residual=big(2), ldr=40) == bad
        assert status(name, residual=big(2) + 64) == bad


def test_route_refusals():
    bad, name = L.ERR_INVALID_ARG, "qgemm_route_topk"
    for change in ({"T": -1}, {"E": 0}, {"E": 1025}, {"k": 0}, {"k": 17}, {"E": 128, "k": 65},
                   {"renormalize": 2}, {"in_dtype": 2}, {"logits": 0}, {"weights": 0},
                   {"experts": 0}, {"offsets": 0}, {"rows": 0}, {"rows": big(2)},
                   {"weights": big(0)}, {"offsets": big(4) + 4}):
        assert status(name, **change) == bad, change
    assert status(name, rows=big(4) + 2) == L.ERR_BAD_ALIGN
    assert status(name, T=0, logits=0, weights=0, experts=0, rows=0) == L.ERR_BAD_HANDLE
    assert status(name, T=1 << 28, E=64, k=8) == L.ERR_UNSUPPORTED


def test_dispatch_and_combine_refusals():
    bad = L.ERR_INVALID_ARG
    for name, w, out in (("qgemm_dispatch_rows", "K", "out"),
                         ("qgemm_dispatch_rows_quantized", "K", "q"),
                         ("qgemm_combine_rows", "N", "out")):
        src = "y" if "combine" in name else "x"
        dt = "dtype" if name == "qgemm_dispatch_rows" else "in_dtype"
        for change in ({"T": -1}, {w: -1}, {"R": -1}, {"k": 0}, {"k": 65}, {dt: 2}, {src: 0},
                       {"rows": 0}, {out: 0}, {out: big(0)}, {out: big(1)}):
            assert status(name, **change) == bad, (name, change)
        assert status(name, rows=big(1) + 1) == L.ERR_BAD_ALIGN
        assert status(name, T=0, **{src: 0, out: 0}) == L.ERR_BAD_HANDLE
        assert status(name, T=1 << 30) == L.ERR_UNSUPPORTED
    assert status("qgemm_dispatch_rows_quantized", sA=0) == bad
    assert status("qgemm_dispatch_rows_quantized", sA=big(2) + 4) == bad
    assert status("qgemm_combine_rows", out_dtype=3) == bad
    assert status("qgemm_combine_rows", out=big(2)) == bad
    assert status("qgemm_combine_rows", residual=big(3)) == L.ERR_BAD_HANDLE
    assert status("qgemm_combine_rows", residual=big(3) + 16) == bad
    assert status("qgemm_combine_rows", weights=0) == L.ERR_BAD_HANDLE


def test_python_names():
    for n in ("linearBf16NK", "w8a8Linear", "expertLinearBf16NK", "w8a8ExpertLinear", "routeTopK",
              "dispatchRows", "dispatchRowsQuantized", "combineRows"):
        assert callable(getattr(qgemm.QuantizedGemmOps, n))
    assert [qgemm.ACT_NONE, qgemm.ACT_RELU, qgemm.ACT_GELU, qgemm.ACT_GELU_TANH,
            qgemm.ACT_SILU] == [0, 1, 2, 3, 4]
    assert ctypes.sizeof(ctypes.c_int) == 4
