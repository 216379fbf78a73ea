"""More rows than a grid has blocks in its second dimension."""
import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("experts", [False, True])
def test_cuda_cores_take_any_number_of_rows(gpu, kind, experts):
    """Rows that the tensor cores cannot take (K = 1), more than 65535 tiles of them.  Small
    integers: the sums are exact, and fp32 holds them."""
    _, st, ops = gpu
    M, N, K = 65535 * 32 + 37, 3, 1
    g = torch.Generator("cuda").manual_seed(3)
    t = torch.bfloat16 if kind == "bf16" else torch.int8
    off = [0, M] if not experts else [0, 5, 5, M - 40, M - 7]
    E = len(off) - 1
    x = torch.randint(-3, 4, (M, K), generator=g, device="cuda").to(t)
    w = torch.randint(-3, 4, (E, N, K), generator=g, device="cuda").to(t)
    out = torch.full((M, N), -77.0, device="cuda")
    o = torch.tensor(off, dtype=torch.int32, device="cuda")
    one, ones = torch.ones(M, device="cuda"), torch.ones(E, N, device="cuda")
    torch.cuda.synchronize()
    if kind == "bf16":
        if experts:
            ops.expertLinearBf16NK(x, w, o, out, E, M, N, K, out_dtype=qgemm.F32)
        else:
            ops.linearBf16NK(x, w, out, M, N, K, out_dtype=qgemm.F32)
    elif experts:
        ops.w8a8ExpertLinear(x, w, one, ones, o, out, E, M, N, K, out_dtype=qgemm.F32)
    else:
        ops.w8a8Linear(x, w, one, ones, out, M, N, K, out_dtype=qgemm.F32)
    st.sync()
    ref = torch.full((M, N), -77.0, device="cuda")
    for e in range(E):
        ref[off[e]:off[e + 1]] = x[off[e]:off[e + 1]].float() @ w[e].float().t()
    assert torch.equal(out, ref)
