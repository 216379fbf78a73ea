"""Sums over very long K: an accumulator that truncates drifts with their length."""
import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [2, 600])
@pytest.mark.parametrize("experts", [False, True])
def test_bf16_outputs_of_very_long_sums(gpu, M, experts):
    """bf16 outputs, K = 2^21: every product is positive, so that an accumulator that truncates
    drifts one way, by 1.9e-3 of the result over all of K in one (half a bf16 step is 2^-8 =
    3.9e-3 of the value at most, 2^-9 at least).  In pieces of 512 values a sum is off by at most
    (32 + 4096) 2^-23 of itself: 32 truncations a piece and the additions of 4096 pieces, each
    half an ulp (2^-24) of a running sum below the whole; then the output's half step."""
    _, st, ops = gpu
    K, N = 1 << 21, 48
    g = torch.Generator("cuda").manual_seed(M)
    x = (torch.rand(M, K, generator=g, device="cuda") + 0.5).bfloat16()
    w = (torch.rand(N, K, generator=g, device="cuda") + 0.5).bfloat16()
    out = torch.empty(M, N, device="cuda").bfloat16()
    off = torch.tensor([0, M], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    if experts:
        ops.expertLinearBf16NK(x, w, off, out, 1, M, N, K, algo=qgemm.ALGO_TCGEN05)
    else:
        ops.linearBf16NK(x, w, out, M, N, K, algo=qgemm.ALGO_TCGEN05)
    st.sync()
    rows = [0, M // 2, M - 1]
    exact = torch.zeros(len(rows), N, dtype=torch.float64, device="cuda")
    for k0 in range(0, K, 1 << 18):
        exact += x[rows, k0:k0 + (1 << 18)].double() @ w[:, k0:k0 + (1 << 18)].double().t()
    drift = (32 * 2.0 ** -23 + 4096 * 2.0 ** -24) * exact
    # the nearest bf16 value of something within `drift` of the exact one
    lo, hi = (exact - drift).bfloat16().double(), (exact + drift).bfloat16().double()
    got = out[rows].double()
    inside = (got >= lo) & (got <= hi)
    assert inside.all(), f"{int((~inside).sum())} of {inside.numel()} outside"


@pytest.mark.parametrize("M,gated", [(2, False), (2, True), (40, True), (300, False), (300, True)])
@pytest.mark.parametrize("experts", [False, True])
def test_bf16_outputs_in_pieces_with_every_epilogue(gpu, M, gated, experts):
    """K = 66048, past where bf16 outputs are summed in pieces; small integers, whose sums are exact
    (9 K < 2^24), so the epilogue's tolerance alone is left."""
    from test_linear_gpu import Case, run
    off = [0, M // 3, M // 3, M] if experts else None
    run(gpu, Case("bf16", M, 203, 66048, act="gelu", gated=gated, bias=True, residual=not experts,
                  offsets=off), qgemm.ALGO_TCGEN05)


@pytest.mark.parametrize("K", [131056, 131071])
def test_int8_sums_at_their_largest(gpu, K):
    """All of x and w at -128: the int32 sum is K 2^14, just below 2^31 (131056 on the tensor cores,
    131071 on CUDA cores); the scales are powers of two, so one rounding to fp32 is left."""
    _, st, ops = gpu
    M, N = 3, 40
    x = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
    w = torch.full((N, K), -128, dtype=torch.int8, device="cuda")
    sx = torch.full((M,), 2.0 ** -10, device="cuda")
    sw = torch.full((N,), 2.0 ** -7, device="cuda")
    out = torch.empty(M, N, device="cuda")
    torch.cuda.synchronize()
    ops.w8a8Linear(x, w, sx, sw, out, M, N, K, out_dtype=qgemm.F32)
    st.sync()
    want = torch.tensor(float(K * 2 ** 14), dtype=torch.float64).float().item() * 2.0 ** -17
    assert (out == want).all()
