"""What an output keeps of its precision through each activation, far out on both sides.

The bounds are those of an evaluation by CUDA's functions, relative to the exact value, with
u = 2^-24 (the half step of fp32), expf within 2 ulp (4 u), erfcf within 4 ulp (8 u), 1 + e and the
quotient within u each:
  silu       v / (1 + exp(-v)): exp's error 4 u, the sum u, the quotient u: 6 u
  gelu       0.5 v erfc(x), x = -v / sqrt 2: the constant and the product err by u each, which
             erfc multiplies by |x erfc'(x) / erfc(x)| <= 2 x^2 + 1 = v^2 + 1 (x > 0; less than 1
             below); erfcf 8 u; two products u each: 2 u (v^2 + 1) + 10 u
  gelu_tanh  v / (1 + exp(-2 w)), w = c (v + d v^3): the two constants, four products and one
             sum err by u each, 7 u at most, doubled argument |2 w| * 7 u; then as silu: 14 |w| u
             + 6 u
plus 2^-126 for results below the normal numbers.  Second-order terms: a factor 1.01.
bf16 outputs add half a bf16 step (2^-8 of the value) and, for silu and gelu_tanh, the fast
exponential's (2 + 1.17 |x|) 2 u of its argument x and the fast quotient's 4 u.
"""
import math

import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]


def reference(act, v):
    """(value, tolerance) in float64."""
    v = v.double()
    if act == "gelu":
        y = 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
        rel = 2 * U * (v * v + 1) + 10 * U
    elif act == "gelu_tanh":
        w = math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
        y = v / (1 + torch.exp(-2 * w))
        rel = 14 * w.abs() * U + 6 * U
    else:
        y = v / (1 + torch.exp(-v))
        rel = torch.full_like(v, 6 * U)
    return y, 1.01 * rel * y.abs() + 2.0 ** -126


# enough rows for each kernel: streamed, its K cut over a cluster, pairs, CUDA cores
FORMS = [(2, 16, 64, qgemm.ALGO_TCGEN05), (2, 2048, 64, qgemm.ALGO_TCGEN05),
         (1500, 256, 2048, qgemm.ALGO_TCGEN05), (3, 16, 64, qgemm.ALGO_SIMT)]


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,K,N,algo", FORMS)
@pytest.mark.parametrize("gated", [False, True])
def test_fp32_outputs_keep_the_activation_to_fp32(gpu, act, M, K, N, algo, gated):
    """The argument comes through the bias alone (the products are zero); a gated layer's up
    half is one."""
    _, st, ops = gpu
    span = {"silu": 80.0, "gelu": 12.0, "gelu_tanh": 9.0}[act]
    v = torch.cat([torch.linspace(-span, span, N - N // 4, device="cuda"),
                   torch.randn(N // 4, generator=torch.Generator("cuda").manual_seed(1),
                               device="cuda")])
    bias = torch.cat([v, torch.ones_like(v)]) if gated else v
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(2 * N if gated else N, K, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(M, N, device="cuda")
    torch.cuda.synchronize()
    ops.linearBf16NK(x, w, out, M, N, K, bias=bias, act=ACTS.index(act), gated=gated,
                     out_dtype=qgemm.F32, algo=algo)
    st.sync()
    y, tol = reference(act, v)
    over = ((out.double() - y).abs() / tol).max(0).values
    at = int(over.argmax())
    assert float(over.max()) <= 1, f"{float(over.max()):.3g} of the tolerance at v = {float(v[at]):.6g}"


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
def test_fp32_outputs_of_int8_experts_keep_the_activation_to_fp32(gpu, act):
    """As above through the int8 experts' kernel."""
    _, st, ops = gpu
    E, M, N, K = 3, 50, 96, 64
    v = torch.linspace(-9, 9, E * N, device="cuda").reshape(E, N)
    off = torch.tensor([0, 20, 20, 50], dtype=torch.int32, device="cuda")
    x = torch.zeros(M, K, dtype=torch.int8, device="cuda")
    w = torch.zeros(E, N, K, dtype=torch.int8, device="cuda")
    s, sw = torch.ones(M, device="cuda"), torch.ones(E, N, device="cuda")
    out = torch.empty(M, N, device="cuda")
    torch.cuda.synchronize()
    ops.w8a8ExpertLinear(x, w, s, sw, off, out, E, M, N, K, bias=v, act=ACTS.index(act),
                         out_dtype=qgemm.F32)
    st.sync()
    y, tol = reference(act, torch.cat([v[0].expand(20, N), v[2].expand(30, N)]))
    assert ((out.double() - y).abs() <= tol).all()


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,K,N,algo", FORMS)
def test_bf16_outputs_are_the_activation_rounded(gpu, act, M, K, N, algo):
    """Relative to each value, the small results of negative arguments among them."""
    _, st, ops = gpu
    span = {"silu": 80.0, "gelu": 12.0, "gelu_tanh": 9.0}[act]
    v = torch.linspace(-span, span, N, device="cuda")
    x = torch.zeros(M, K, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(N, K, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(M, N, device="cuda").bfloat16()
    torch.cuda.synchronize()
    ops.linearBf16NK(x, w, out, M, N, K, bias=v, act=ACTS.index(act), algo=algo)
    st.sync()
    y, tol = reference(act, v)
    if act != "gelu":
        arg = v.double().abs()
        if act == "gelu_tanh":
            arg = 2 * math.sqrt(2 / math.pi) * (arg + 0.044715 * arg ** 3)
        tol = tol + 1.01 * ((2 + 1.17 * arg) * 2 * U + 4 * U) * y.abs()
    tol = tol + 2.0 ** -8 * (y.abs() + tol)
    assert ((out.double() - y).abs() <= tol).all()
