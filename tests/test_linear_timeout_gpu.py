"""The linear layers' way out when a wait runs out, taken on purpose and without a fault: with the
hold-back hook their epilogues wait, bounded, for what never comes, while copies and MMAs go on.
The kernel gives up, waits for what it has under way, reports the timeout and ends; the same
stream then runs the same layer right."""
import pytest

import qgemm
from test_linear_gpu import Case

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

OFF = [0, 3, 3, 200, 210, 470, 600]
CASES = {  # each kernel, with few and with many tiles a CTA
    "streamed": ("bf16", 5, 20002, 1040, dict(bias=True)),
    "streamed, K cut": ("bf16", 1, 4096, 4096, dict(residual=True)),
    "streamed, K cut, gated int8": ("w8a8", 33, 1000, 4096, dict(gated=True, act="silu")),
    "streamed, fp32 in pieces": ("bf16", 40, 9000, 2048, dict(out="f32")),
    "pairs": ("bf16", 600, 2304, 2048, dict(bias=True, act="gelu")),
    "pairs, many tiles": ("w8a8", 4096, 4096, 2048, dict(residual=True)),
    "pairs, fp32 in pieces": ("bf16", 2048, 2304, 2048, dict(out="f32")),
    "experts": ("w8a8", 600, 1000, 1024, dict(gated=True, act="silu", offsets=OFF)),
    "experts, many rows": ("bf16", 6000, 520, 2048, dict(offsets=[10 * o for o in OFF])),
}


@pytest.mark.parametrize("name", sorted(CASES))
def test_a_wait_that_runs_out_ends_the_call_and_the_stream_goes_on(gpu, name):
    dev, _, _ = gpu
    kind, M, N, K, more = CASES[name]
    c = Case(kind, M, N, K, **more)
    st = dev.stream()
    ops = qgemm.QuantizedGemmOps(st)
    old = dev.wait_limit_ns
    dev.wait_limit_ns = 20_000_000
    dev.debug_hold_split(True)
    try:
        c.call(ops, qgemm.ALGO_TCGEN05)
        with pytest.raises(qgemm.QGemmError) as e:
            st.sync()
        assert e.value.status == qgemm._lib.ERR_TIMEOUT
        assert (c.buf == -77.25).all()   # a layer that gave up has stored nothing
    finally:
        dev.debug_hold_split(False)
        dev.wait_limit_ns = old
    st.sync()   # reported once
    for _ in range(2):
        c.call(ops, qgemm.ALGO_TCGEN05)
        st.sync()
        c.check()
    st.destroy()


@pytest.mark.parametrize("name", sorted(CASES))
@pytest.mark.parametrize("limit", [1000, 4000])
def test_limits_shorter_than_a_copy(gpu, name, limit):
    """A limit of a few microseconds runs out in any wait, at any point, in one CTA of a pair or
    cluster before the other: the call ends all the same, and is right or reported."""
    dev, _, _ = gpu
    kind, M, N, K, more = CASES[name]
    c = Case(kind, M, N, K, **more)
    st = dev.stream()
    ops = qgemm.QuantizedGemmOps(st)
    old = dev.wait_limit_ns
    for _ in range(3):
        c.out.fill_(-77.25)
        torch.cuda.synchronize()
        dev.wait_limit_ns = limit
        try:
            c.call(ops, qgemm.ALGO_TCGEN05)
            try:
                st.sync()
                c.check()
            except qgemm.QGemmError as e:
                assert e.status == qgemm._lib.ERR_TIMEOUT
        finally:
            dev.wait_limit_ns = old
        st.sync()
    c.out.fill_(-77.25)
    torch.cuda.synchronize()
    c.call(ops, qgemm.ALGO_TCGEN05)
    st.sync()
    c.check()
    st.destroy()
