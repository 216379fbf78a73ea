"""Who learns of a bad offset or row index: the stream handle that made the call, at its next
sync, and nobody else; and a wait that ran out is reported beside it, not hidden by it."""
import numpy as np
import pytest

import qgemm
import qgemm.synthetic as syn
from helpers import Out, dev_array

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def bad_combine(ops, R=4):
    """A combine whose second pair names a row past the last."""
    y = torch.ones(R, 64, device="cuda").bfloat16()
    rows = torch.tensor([[0, R]], dtype=torch.int32, device="cuda")
    out = torch.empty(1, 64, device="cuda").bfloat16()
    torch.cuda.synchronize()
    ops.combineRows(y, rows, None, out, 1, 2, 64, R)
    return y, rows, out


def bad_linear(ops, algo):
    x = torch.ones(8, 64, device="cuda").bfloat16()
    w = torch.ones(2, 32, 64, device="cuda").bfloat16()
    off = torch.tensor([0, 4, 9], dtype=torch.int32, device="cuda")
    out = torch.empty(8, 32, device="cuda").bfloat16()
    torch.cuda.synchronize()
    ops.expertLinearBf16NK(x, w, off, out, 2, 8, 32, 64, algo=algo)
    return x, w, off, out


def bad_dispatch(ops, quantised):
    x = torch.ones(1, 64, device="cuda").bfloat16()
    rows = torch.tensor([[0, 9]], dtype=torch.int32, device="cuda")
    q = torch.empty(9, 64, dtype=torch.int8 if quantised else torch.bfloat16, device="cuda")
    s = torch.empty(9, device="cuda")
    torch.cuda.synchronize()
    if quantised:
        ops.dispatchRowsQuantized(x, rows, q, s, 1, 2, 64, 9)
    else:
        ops.dispatchRows(x, rows, q, 1, 2, 64, 9)
    return x, rows, q, s


CALLS = {"combine": bad_combine, "dispatch": lambda o: bad_dispatch(o, False),
         "dispatch quantised": lambda o: bad_dispatch(o, True),
         "experts": lambda o: bad_linear(o, qgemm.ALGO_TCGEN05),
         "experts, CUDA cores": lambda o: bad_linear(o, qgemm.ALGO_SIMT)}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_the_stream_that_called_is_told_and_no_other(gpu, name):
    dev, _, _ = gpu
    a, b = dev.stream(), dev.stream()
    try:
        keep = CALLS[name](qgemm.QuantizedGemmOps(a))
        torch.cuda.synchronize()
        b.sync()
        with pytest.raises(qgemm.QGemmError) as e:
            a.sync()
        assert e.value.status == qgemm._lib.ERR_INVALID_ARG
        a.sync()
        b.sync()
        del keep
    finally:
        a.destroy()
        b.destroy()


def test_a_bad_index_does_not_hide_a_wait_that_ran_out(gpu):
    """A combine with a bad row, then a GEMM whose split waits run out (the hold-back hook): one
    sync reports the timeout, the next the index."""
    dev, _, _ = gpu
    st = dev.stream()
    ops = qgemm.QuantizedGemmOps(st)
    M, N, K = 3840, 4096, 1024
    A, B, sA, sB = syn.w8a8_inputs(M, N, K, seed=77)
    dA, dB, dsA, dsB = (dev_array(gpu, a) for a in (A, B, sA, sB))
    y = Out(dev, st, M * N * 2)
    st.sync()
    old = dev.wait_limit_ns
    dev.wait_limit_ns = 20_000_000
    dev.debug_hold_split(True)
    try:
        keep = bad_combine(ops)
        ops.w8a8Gemm(dA, dB, dsA, dsB, y, M, N, K, algo=qgemm.ALGO_TCGEN05)
        got = []
        for _ in range(2):
            with pytest.raises(qgemm.QGemmError) as e:
                st.sync()
            got.append(e.value.status)
        assert got == [qgemm._lib.ERR_TIMEOUT, qgemm._lib.ERR_INVALID_ARG]
        del keep
    finally:
        dev.debug_hold_split(False)
        dev.wait_limit_ns = old
    st.sync()
    ops.w8a8Gemm(dA, dB, dsA, dsB, y, M, N, K, algo=qgemm.ALGO_TCGEN05)
    st.sync()
    st.destroy()


def test_many_stream_handles_keep_their_errors_apart(gpu):
    """Handles come and go: a new one starts clean, whatever the one before it left unread."""
    dev, _, _ = gpu
    for _ in range(50):
        a = dev.stream()
        keep = bad_combine(qgemm.QuantizedGemmOps(a))
        torch.cuda.synchronize()
        a.destroy()
        b = dev.stream()
        b.sync()
        b.destroy()
        del keep
    held = [dev.stream() for _ in range(64)]
    try:
        keep = bad_combine(qgemm.QuantizedGemmOps(held[37]))
        torch.cuda.synchronize()
        told = []
        for i, st in enumerate(held):
            try:
                st.sync()
            except qgemm.QGemmError as e:
                assert e.status == qgemm._lib.ERR_INVALID_ARG
                told.append(i)
        assert told == [37]
        assert np.isfinite(float(keep[2].float().sum()))
    finally:
        for st in held:
            st.destroy()


def test_more_handles_than_words(gpu):
    """Past 4095 handles at a time the last word is shared: errors still reach the handle that
    called, if it is the next of them to be synchronised."""
    dev, _, _ = gpu
    own = dev.stream()
    raw = torch.cuda.Stream().cuda_stream
    held = [dev.wrap_stream(raw) for _ in range(4200)]
    try:
        for i in (10, 4199):
            keep = bad_combine(qgemm.QuantizedGemmOps(held[i]))
            torch.cuda.synchronize()
            own.sync()
            with pytest.raises(qgemm.QGemmError):
                held[i].sync()
            held[i].sync()
            del keep
    finally:
        for st in held:
            st.destroy()
    own.destroy()
    st = dev.stream()
    st.sync()
    st.destroy()
