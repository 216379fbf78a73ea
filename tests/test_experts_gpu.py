"""ExpertMLP: the routing, dispatch, expert and combine calls run together, as a serving program
runs them.  Every stage is checked against its definition on the values that the stage before
left on the device (so roundings do not pile up in the comparison), then the whole is captured
into a graph and replayed on new tokens.

Tolerances: logits, 48 units of the fp32 accumulator (2^-23) of sum |x w| for K = 512 values an
accumulator piece plus the pieces (K = 1024 here: 2 pieces); expert layers as in
test_linear_gpu (int32 sums are exact; SiLU's own error; half a bf16 step); combine k products."""
import numpy as np
import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E, K_TOP, H, F = 8, 2, 1024, 1408


def view(buf, dtype, shape):
    """A torch copy of a qgemm buffer."""
    st, n = view.st, int(np.prod(shape))
    itemsize = torch.empty((), dtype=dtype).element_size()
    raw = buf.to_numpy(st, np.uint8, (buf.nbytes,))[:n * itemsize]
    return torch.from_numpy(raw.copy()).view(dtype).reshape(shape).cuda()


@pytest.fixture(scope="module")
def layer(gpu):
    dev, st, ops = gpu
    view.st = st
    g = torch.Generator("cuda").manual_seed(11)
    router = (torch.randn(E, H, generator=g, device="cuda") * H ** -0.5).bfloat16()
    w1 = torch.randint(-127, 128, (E, 2 * F, H), generator=g, device="cuda", dtype=torch.int8)
    w2 = torch.randint(-127, 128, (E, H, F), generator=g, device="cuda", dtype=torch.int8)
    s1 = (torch.rand(E, 2 * F, generator=g, device="cuda") + 0.5) / (73 * H ** 0.5)
    s2 = (torch.rand(E, H, generator=g, device="cuda") + 0.5) / (73 * F ** 0.5)
    torch.cuda.synchronize()
    mlp = qgemm.ExpertMLP(ops, router, w1, s1, w2, s2, E=E, k=K_TOP, H=H, F=F, max_tokens=700)
    yield mlp
    st.sync()
    mlp.close()


def check(mlp, x, out, residual, T):
    R = T * K_TOP
    xd = x.double()
    logits = view(mlp.logits, torch.float32, (T, E))
    ref = xd @ mlp.router.double().t()
    assert ((logits.double() - ref).abs() <= 48 * 2 ** -23 * (xd.abs() @ mlp.router.double().abs().t())).all()
    # routing, from the logits on the device
    experts = view(mlp.experts, torch.int32, (T, K_TOP))
    want = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :K_TOP]
    assert torch.equal(experts.long(), want)
    off = view(mlp.offsets, torch.int32, (E + 1,)).tolist()
    rows = view(mlp.rows, torch.int32, (T, K_TOP)).long()
    flat = experts.reshape(-1).long()
    order = torch.sort(flat, stable=True).indices
    pos = torch.empty_like(flat)
    pos[order] = torch.arange(R, device="cuda")
    assert torch.equal(rows.reshape(-1), pos)
    assert off == [0] + torch.cumsum(torch.bincount(flat, minlength=E), 0).tolist()
    # dispatch: the per-token quantiser's values
    xq, sx = view(mlp.xq, torch.int8, (R, H)), view(mlp.sx, torch.float32, (R,))
    f = x.float()
    most = f.abs().amax(1)
    full = torch.full_like(most, 127.0)
    q = torch.clamp(torch.trunc(f * (full / most)[:, None]), -128, 127).to(torch.int8)
    for j in range(K_TOP):
        assert torch.equal(xq[rows[:, j]], q)
        assert torch.equal(sx[rows[:, j]], most / full)
    # the experts' layers
    h = view(mlp.h, torch.bfloat16, (R, F)).double()
    hq, sh = view(mlp.hq, torch.int8, (R, F)), view(mlp.sh, torch.float32, (R,))
    y = view(mlp.y, torch.bfloat16, (R, H)).double()
    for e in range(E):
        a, b = off[e], off[e + 1]
        if a == b:
            continue
        z = (xq[a:b].double() @ mlp.w1[e].double().t()) * mlp.s1[e].double() * sx[a:b].double()[:, None]
        ez = 2 * U * z.abs()
        gate, up = z[:, :F], z[:, F:]
        act = gate * torch.sigmoid(gate)
        ea = 1.2 * ez[:, :F] + 2 * U * (8 + 1.2 * gate.abs()) * act.abs()
        ref = act * up
        tol = ea * up.abs() + act.abs() * ez[:, F:] + 2 * U * ref.abs()
        tol = tol + 2.0 ** -8 * (ref.abs() + tol)
        assert ((h[a:b] - ref).abs() <= tol).all()
        ref = (hq[a:b].double() @ mlp.w2[e].double().t()) * mlp.s2[e].double() * sh[a:b].double()[:, None]
        assert ((y[a:b] - ref).abs() <= (2.0 ** -8 + 4 * U) * ref.abs()).all()
    w = view(mlp.weights, torch.float32, (T, K_TOP)).double()
    parts = w[:, :, None] * y[rows]
    ref = parts.sum(1) + (residual.double() if residual is not None else 0)
    tol = 4 * U * (parts.abs().sum(1) + ref.abs())
    assert ((out.double() - ref).abs() <= tol + 2.0 ** -8 * (ref.abs() + tol)).all()


@pytest.mark.parametrize("T", [1, 2, 7, 33, 256, 257, 700])
@pytest.mark.parametrize("with_residual", [False, True])
def test_expert_mlp(gpu, layer, T, with_residual):
    _, st, _ = gpu
    g = torch.Generator("cuda").manual_seed(T)
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    residual = torch.randn(T, H, generator=g, device="cuda").bfloat16() if with_residual else None
    out = torch.full((T + 1, H), 9.0, device="cuda").bfloat16()
    torch.cuda.synchronize()
    layer(x, out, T, residual=residual)
    st.sync()
    check(layer, x, out[:T], residual, T)
    assert (out[T] == 9.0).all()


def test_expert_mlp_adds_onto_its_input(gpu, layer):
    """The block's usual form: x += layer(x)."""
    _, st, _ = gpu
    x = torch.randn(50, H, device="cuda").bfloat16()
    apart = torch.empty_like(x)
    torch.cuda.synchronize()
    layer(x, apart, 50, residual=x)
    layer(x, x, 50, residual=x)
    st.sync()
    assert torch.equal(x, apart)


def test_expert_mlp_captured(gpu, layer):
    dev, _, _ = gpu
    T = 40
    side = torch.cuda.Stream()
    st = dev.wrap_stream(side.cuda_stream)
    mlp = qgemm.ExpertMLP(qgemm.QuantizedGemmOps(st), layer.router, layer.w1, layer.s1, layer.w2,
                          layer.s2, E=E, k=K_TOP, H=H, F=F, max_tokens=T)
    x = torch.randn(T, H, device="cuda").bfloat16()
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    mlp(x, out, T)
    st.sync()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        mlp(x, out, T)
    for i in range(3):
        x.copy_(torch.randn(T, H, device="cuda") * (i + 1))
        out.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.zero_()
        torch.cuda.synchronize()
        mlp(x, out, T)
        st.sync()
        assert torch.equal(out, got)
        check(mlp, x, out, None, T)
    del graph
    mlp.close()
    st.destroy()


def test_expert_mlp_refuses_more_tokens_than_it_holds(gpu, layer):
    with pytest.raises(ValueError):
        layer(0, 0, 701)
    layer(0, 0, 0)
