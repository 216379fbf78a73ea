"""Routing, dispatch and combine on the GPU, against their definitions.

Whole numbers (experts, offsets, rows, copied rows, int8 values) are compared for equality.
Weights: exp and the sum's additions and the quotient in fp32, against float64: the exponent's
argument l - max carries one rounding of |l - max| (up to |l - max| u in exp), expf 2 ulp, the
sum of at most E terms log2-deep over lanes plus E / 32 serial additions, the quotient half an
ulp: (8 + E / 32 + |l - max|) 2^-23 relative.  Combine: k products and sums, each within u of
the sum of magnitudes, then the residual's addition and the output's half step.
"""
import numpy as np
import pytest

import qgemm
import qgemm.synthetic as syn
from helpers import Out, dev_array

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def route_ref(v, k):
    """experts, rows, offsets of float64 logits v: largest first, ties to the lower index."""
    T, E = v.shape
    experts = np.full((T, k), -1, np.int32)
    for t in range(T):
        ok = [e for e in range(E) if v[t, e] > -np.inf]  # NaN compares false
        ok.sort(key=lambda e: (-v[t, e], e))
        experts[t, :min(k, len(ok))] = ok[:k]
    rows = np.full(T * k, -1, np.int32)
    flat = experts.reshape(-1)
    order = np.argsort(flat, kind="stable")
    order = order[flat[order] >= 0]
    rows[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=E))])
    return experts, rows.reshape(T, k), offsets.astype(np.int32)


def route(gpu, logits, k, renormalize=True, dtype="f32"):
    dev, st, ops = gpu
    T, E = logits.shape
    h = logits.astype(np.float32) if dtype == "f32" else syn.bf16_bits(logits)
    w, e = Out(dev, st, T * k * 4), Out(dev, st, T * k * 4)
    o, r = Out(dev, st, (E + 1) * 4), Out(dev, st, T * k * 4)
    ops.routeTopK(dev_array(gpu, h), w, e, o, r, T, E, k, renormalize=renormalize,
                  in_dtype=qgemm.F32 if dtype == "f32" else qgemm.BF16)
    st.sync()
    v = h.astype(np.float64) if dtype == "f32" else syn.bf16_to_float(h).astype(np.float64)
    return (w.read(np.float32, (T, k)), e.read(np.int32, (T, k)), o.read(np.int32, (E + 1,)),
            r.read(np.int32, (T, k)), v)


def check_route(gpu, logits, k, renormalize=True, dtype="f32"):
    w, e, o, r, v = route(gpu, logits, k, renormalize, dtype)
    experts, rows, offsets = route_ref(v, k)
    np.testing.assert_array_equal(e, experts)
    np.testing.assert_array_equal(o, offsets)
    np.testing.assert_array_equal(r, rows)
    T, E = v.shape
    for t in range(T):
        ok = experts[t] >= 0
        assert (w[t][~ok] == 0).all()
        if not ok.any():
            continue
        top = np.minimum(v[t][experts[t][ok]], np.finfo(np.float32).max)
        every = np.where(np.isnan(v[t]), -np.inf, np.minimum(v[t], np.finfo(np.float32).max))
        over = top if renormalize else every
        p = np.exp(top - top[0]) / np.exp(over - top[0]).sum()
        tol = (8 + E / 32 + np.minimum(np.abs(top - top[0]), 200.)) * 2 * U * p + 1e-37
        assert (np.abs(w[t][ok] - p) <= tol).all()


@pytest.mark.parametrize("T,E,k", [
    (1, 1, 1), (1, 8, 2), (3, 4, 4), (16, 8, 2), (32, 64, 8), (33, 60, 6), (70, 33, 1),
    (257, 128, 8), (512, 64, 8), (513, 8, 2), (700, 256, 8), (1500, 100, 3), (40, 1024, 64),
    (600, 1024, 33)])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route(gpu, T, E, k, renormalize):
    rng = np.random.default_rng(T + E + k)
    check_route(gpu, rng.standard_normal((T, E)) * 2, k, renormalize,
                "bf16" if (T + E) % 2 else "f32")


@pytest.mark.parametrize("T", [5, 300, 800])
def test_route_ties_go_to_the_lower_index(gpu, T):
    rng = np.random.default_rng(T)
    check_route(gpu, rng.integers(-1, 2, (T, 40)).astype(np.float64), 6)
    check_route(gpu, np.zeros((T, 70)), 7)
    signed = np.where(rng.random((T, 9)) < 0.5, 0.0, -0.0)   # equal, whatever their sign
    check_route(gpu, signed, 3)


@pytest.mark.parametrize("T", [4, 600])
@pytest.mark.parametrize("renormalize", [True, False])
def test_route_masked_experts(gpu, T, renormalize):
    """-inf and NaN are never chosen, the type's lowest value is (last); rows with nothing left
    route nowhere; +inf counts as the largest finite value."""
    rng = np.random.default_rng(T)
    v = rng.standard_normal((T, 12))
    v[rng.random(v.shape) < 0.5] = -np.inf
    v[rng.random(v.shape) < 0.1] = np.nan
    v[1] = -np.inf
    v[2] = np.nan
    v[3, :] = -np.inf
    v[3, 7] = np.finfo(np.float32).min
    check_route(gpu, v, 4, renormalize)
    u = rng.standard_normal((T, 12))
    u[0, 3] = u[0, 9] = np.inf
    u[1, :] = np.finfo(np.float32).min
    u[2, 5] = np.finfo(np.float32).max
    check_route(gpu, u, 3, renormalize)


def test_route_no_tokens_and_one_expert_for_all(gpu):
    dev, st, ops = gpu
    o = Out(dev, st, 9 * 4)
    ops.routeTopK(0, 0, 0, o, 0, 0, 8, 2)
    st.sync()
    assert (o.read(np.int32, (9,)) == 0).all()
    v = np.zeros((900, 16))
    v[:, 11] = 5
    check_route(gpu, v, 1)


def test_route_large_is_a_stable_sort(gpu):
    """131072 pairs: offsets and rows against numpy's stable sort of the experts it chose."""
    dev, st, ops = gpu
    T, E, k = 16384, 64, 8
    rng = np.random.default_rng(0)
    h = rng.standard_normal((T, E)).astype(np.float32)
    w, e, o, r, _ = route(gpu, h, k, False)
    want = np.argsort(-h, axis=1, kind="stable")[:, :k]
    np.testing.assert_array_equal(e, want)
    flat = e.reshape(-1)
    rows = np.empty(T * k, np.int32)
    rows[np.argsort(flat, kind="stable")] = np.arange(T * k)
    np.testing.assert_array_equal(r.reshape(-1), rows)
    np.testing.assert_array_equal(o, np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=E))]))


# ---- dispatch ------------------------------------------------------------------------------

def random_rows(T, k, R, rng, drop=0.1):
    rows = rng.permutation(R)[:T * k].astype(np.int32)
    rows[rng.random(T * k) < drop] = -1
    return rows.reshape(T, k)


@pytest.mark.parametrize("T,k,K", [(1, 1, 8), (1, 8, 4096), (5, 2, 13), (33, 2, 4096),
                                   (64, 6, 1000), (7, 3, 8200), (300, 4, 1), (9, 2, 12000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_dispatch_copy_and_quantised(gpu, oracle, T, k, K, dtype):
    dev, st, ops = gpu
    rng = np.random.default_rng(T * k + K)
    R = T * k + 3
    rows = random_rows(T, k, R, rng)
    x = rng.standard_normal((T, K)).astype(np.float32)
    x[0] = 0
    h = x if dtype == "f32" else syn.bf16_bits(x)
    code = qgemm.F32 if dtype == "f32" else qgemm.BF16
    out = Out(dev, st, R * K * h.itemsize)
    xd, rd = dev_array(gpu, h), dev_array(gpu, rows)
    ops.dispatchRows(xd, rd, out, T, k, K, R, dtype=code)
    q, s = Out(dev, st, R * K), Out(dev, st, R * 4)
    ops.dispatchRowsQuantized(xd, rd, q, s, T, k, K, R, in_dtype=code)
    # the sibling on the same tokens: the same values and scales
    q0, s0 = Out(dev, st, T * K), Out(dev, st, T * 4)
    ops.quantizePerToken(xd, q0, s0, T, K, in_dtype=code)
    st.sync()
    got, gq, gs = out.read(h.dtype, (R, K)), q.read(np.int8, (R, K)), s.read(np.float32, (R,))
    q0, s0 = q0.read(np.int8, (T, K)), s0.read(np.float32, (T,))
    hit = np.zeros(R, bool)
    for t in range(T):
        for r in rows[t]:
            if r >= 0:
                hit[r] = True
                np.testing.assert_array_equal(got[r], h[t])
                np.testing.assert_array_equal(gq[r], q0[t])
                assert gs[r] == s0[t]
    assert (got[~hit].view(np.uint8) == 0xA5).all()     # rows of no pair stay as they were
    assert (gq[~hit].view(np.uint8) == 0xA5).all()
    assert (gs[~hit].view(np.uint8) == 0xA5).all()


def test_dispatch_quantised_nan_and_infinity(gpu):
    """A NaN never becomes the maximum and quantises to 0; an infinity takes the row with it as
    in quantizePerToken (whose result it must be)."""
    dev, st, ops = gpu
    x = np.random.default_rng(1).standard_normal((4, 64)).astype(np.float32)
    x[1, 5] = np.nan
    x[2, 7] = np.inf
    x[3, :] = np.nan
    rows = np.arange(4, dtype=np.int32)[::-1].copy()
    q, s = Out(dev, st, 4 * 64), Out(dev, st, 16)
    q0, s0 = Out(dev, st, 4 * 64), Out(dev, st, 16)
    xd = dev_array(gpu, x)
    ops.dispatchRowsQuantized(xd, dev_array(gpu, rows), q, s, 4, 1, 64, 4, in_dtype=qgemm.F32)
    ops.quantizePerToken(xd, q0, s0, 4, 64, in_dtype=qgemm.F32)
    st.sync()
    np.testing.assert_array_equal(q.read(np.int8, (4, 64))[::-1], q0.read(np.int8, (4, 64)))
    np.testing.assert_array_equal(s.read(np.uint32, (4,))[::-1], s0.read(np.uint32, (4,)))


def test_rows_out_of_range_are_skipped_and_reported(gpu):
    dev, st, ops = gpu
    T, k, K, R = 6, 2, 64, 12
    rng = np.random.default_rng(2)
    x = syn.bf16_bits(rng.standard_normal((T, K)).astype(np.float32))
    rows = np.arange(T * k, dtype=np.int32).reshape(T, k)
    rows[2, 1] = R
    rows[4, 0] = 2 ** 31 - 1
    xd, rd = dev_array(gpu, x), dev_array(gpu, rows)
    out, q, s = Out(dev, st, R * K * 2), Out(dev, st, R * K), Out(dev, st, R * 4)
    y, o = dev_array(gpu, np.zeros((R, K), np.uint16)), Out(dev, st, T * K * 2)
    for call in (lambda: ops.dispatchRows(xd, rd, out, T, k, K, R),
                 lambda: ops.dispatchRowsQuantized(xd, rd, q, s, T, k, K, R),
                 lambda: ops.combineRows(y, rd, None, o, T, k, K, R)):
        call()
        with pytest.raises(qgemm.QGemmError) as e:
            st.sync()
        assert e.value.status == qgemm._lib.ERR_INVALID_ARG
        st.sync()
    got = out.read(np.uint16, (R, K))
    for t in range(T):
        for j in range(k):
            if rows[t, j] < R:
                np.testing.assert_array_equal(got[rows[t, j]], x[t])
    assert (got[[5, 8]].view(np.uint8) == 0xA5).all()
    assert (o.read(np.uint16, (T, K)) == 0).all()


# ---- combine -------------------------------------------------------------------------------

@pytest.mark.parametrize("T,k,N", [(1, 1, 8), (1, 2, 4096), (16, 2, 4096), (5, 8, 1000), (33, 6, 13),
                                   (300, 4, 264), (3, 64, 40), (9, 5, 2056)])
@pytest.mark.parametrize("ti", ["bf16", "f32"])
@pytest.mark.parametrize("to", ["bf16", "f32"])
def test_combine(gpu, T, k, N, ti, to):
    _, st, ops = gpu
    g = torch.Generator("cuda").manual_seed(T + k + N)
    dt = {"bf16": torch.bfloat16, "f32": torch.float32}
    code = {"bf16": qgemm.BF16, "f32": qgemm.F32}
    R = T * k + 2
    rows = torch.from_numpy(random_rows(T, k, R, np.random.default_rng(T))).cuda()
    y = torch.randn((R, N), generator=g, device="cuda").to(dt[ti])
    named = torch.zeros(R, dtype=torch.bool, device="cuda")
    named[rows[rows >= 0].long()] = True
    y[~named] = float("nan")    # a row of no pair is never read into a sum
    w = torch.randn((T, k), generator=g, device="cuda")
    res = torch.randn((T, N), generator=g, device="cuda").to(dt[to])
    for weights, residual in ((w, res), (w, None), (None, res)):
        buf = torch.full((T * N + 32,), 3.5, dtype=dt[to], device="cuda")
        out = buf[16:16 + T * N].view(T, N)
        torch.cuda.synchronize()
        ops.combineRows(y, rows, weights, out, T, k, N, R, residual=residual, in_dtype=code[ti],
                        out_dtype=code[to])
        st.sync()
        safe = rows.clamp_min(0).long()
        yy = torch.where((rows >= 0)[:, :, None], y[safe].double(), torch.zeros((), dtype=torch.float64, device="cuda"))
        ww = (weights if weights is not None else torch.ones_like(w)).double()[:, :, None]
        ref = (ww * yy).sum(1)
        mag = (ww * yy).abs().sum(1)
        if residual is not None:
            ref = ref + residual.double()
        tol = k * U * mag * 1.01 + U * ref.abs()
        tol = tol + (2.0 ** -8 if to == "bf16" else U) * (ref.abs() + tol)
        assert ((out.double() - ref).abs() <= tol).all()
        assert (buf[:16] == 3.5).all() and (buf[16 + T * N:] == 3.5).all()


def test_combine_onto_the_residual_in_place(gpu):
    _, st, ops = gpu
    T, k, N = 40, 2, 520
    rows = torch.arange(T * k, dtype=torch.int32, device="cuda").view(T, k)
    y = torch.randn(T * k, N, device="cuda").bfloat16()
    w = torch.rand(T, k, device="cuda")
    x = torch.randn(T, N, device="cuda").bfloat16()
    apart = torch.empty_like(x)
    torch.cuda.synchronize()
    ops.combineRows(y, rows, w, apart, T, k, N, T * k, residual=x)
    ops.combineRows(y, rows, w, x, T, k, N, T * k, residual=x)
    st.sync()
    assert torch.equal(x, apart)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_route_infinity_beats_the_largest_finite_value(gpu, dtype):
    """+inf counts as the largest finite fp32: above bf16's largest, equal to fp32's own."""
    big = 3.3895313892515355e38  # bf16's largest
    v = np.zeros((70, 20))
    v[:, 4] = big
    v[:, 11] = np.inf
    v[3, 11] = -np.inf
    check_route(gpu, v, 3, True, dtype)
    check_route(gpu, v, 3, False, dtype)
