"""The tensor-core GEMM kernels under wait limits shorter than a copy: a wait runs out at any point,
in one CTA of a pair before the other.  The call ends, after what it has under way, with the right
result or a reported timeout, and the next call on the stream is right."""
import numpy as np
import pytest

import qgemm
import qgemm.synthetic as syn
from helpers import Out, dev_array

pytestmark = pytest.mark.gpu


def w8a8(gpu, M, N, K):
    A, B, sA, sB = syn.w8a8_inputs(M, N, K, seed=M + N + K)
    d = [dev_array(gpu, a) for a in (A, B, sA, sB)]
    return (lambda ops, y: ops.w8a8Gemm(*d, y, M, N, K, algo=qgemm.ALGO_TCGEN05)), M * N * 2


def bf16(gpu, M, N, K):
    rng = np.random.default_rng(M + N + K)
    d = [dev_array(gpu, syn.bf16_bits(rng.standard_normal(s).astype(np.float32))) for s in ((M, K), (N, K))]
    return (lambda ops, y: ops.gemmBf16NK(*d, y, M, N, K)), M * N * 2


def f32(gpu, M, N, K):
    rng = np.random.default_rng(M + N + K)
    d = [dev_array(gpu, rng.standard_normal(s).astype(np.float32)) for s in ((M, K), (K, N))]
    return (lambda ops, y: qgemm.MatrixOps(ops.stream).gemmF32(*d, y, M, N, K, algo=qgemm.ALGO_TCGEN05)), M * N * 4


def prefill(gpu, M, N, K):
    dev, st, ops = gpu
    x, wq, sc = syn.w4a16_inputs(M, N, K, group=128, seed=M + N + K)
    wf = Out(dev, st, ops.w4FragBytes(K, N))
    ops.prepackW4Frag(dev_array(gpu, wq), wf, K, N)
    dx, ds = dev_array(gpu, x), dev_array(gpu, sc)
    n = ops.w4PrefillWorkspaceBytes(K, N)
    ws = Out(dev, st, n)
    st.sync()
    return (lambda o, y: o.w4a16GemmGroupedPrefillFrag(dx, wf, ds, y, M, N, K, ws, n)), M * N * 2


CASES = {"w8a8, one CTA a tile": (w8a8, 128, 4096, 4096), "w8a8, split tail": (w8a8, 3840, 4096, 1024),
         "w8a8, pairs": (w8a8, 2048, 2304, 4096), "bf16": (bf16, 512, 1024, 4096),
         "fp32": (f32, 512, 1024, 1024), "group-scaled prefill": (prefill, 2048, 4096, 4096)}


@pytest.mark.parametrize("name", sorted(CASES))
@pytest.mark.parametrize("limit", [1000, 4000, 20000])
def test_limits_shorter_than_a_copy(gpu, name, limit):
    dev, st0, _ = gpu
    make, M, N, K = CASES[name]
    call, nbytes = make(gpu, M, N, K)
    st0.sync()
    st = dev.stream()
    ops = qgemm.QuantizedGemmOps(st)
    y = Out(dev, st, nbytes)
    call(ops, y)
    st.sync()
    want = y.read(np.uint8, (nbytes,)).copy()
    old = dev.wait_limit_ns
    for _ in range(3):
        st.memset(y.address, 0, nbytes)
        st.sync()
        dev.wait_limit_ns = limit
        try:
            call(ops, y)
            try:
                st.sync()
                np.testing.assert_array_equal(y.read(np.uint8, (nbytes,)), want)
            except qgemm.QGemmError as e:
                assert e.status == qgemm._lib.ERR_TIMEOUT
        finally:
            dev.wait_limit_ns = old
        st.sync()
        call(ops, y)
        st.sync()
        np.testing.assert_array_equal(y.read(np.uint8, (nbytes,)), want)
    st.destroy()
