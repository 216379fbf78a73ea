"""Operands, residual and output as columns of one wider buffer: the same bits as apart, and
nothing beside the output's columns is touched."""
import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 3, 40, 600])
@pytest.mark.parametrize("algo", [qgemm.ALGO_TCGEN05, qgemm.ALGO_SIMT])
@pytest.mark.parametrize("gated", [False, True])
def test_columns_of_one_buffer(gpu, M, algo, gated):
    _, st, ops = gpu
    K, N, ld = 256, 100, 512
    g = torch.Generator("cuda").manual_seed(M)
    buf = torch.randn(M, ld, generator=g, device="cuda").bfloat16()
    x, res, out = buf[:, :K], buf[:, K:K + N], buf[:, K + N:K + 2 * N]
    w = torch.randn(2 * N if gated else N, K, generator=g, device="cuda").bfloat16()
    apart = torch.empty(M, N, device="cuda").bfloat16()
    kept, xc, rc = buf.clone(), x.contiguous(), res.contiguous()
    torch.cuda.synchronize()
    kw = dict(act=qgemm.ACT_SILU, gated=gated, algo=algo)
    ops.linearBf16NK(xc, w, apart, M, N, K, residual=rc, **kw)
    ops.linearBf16NK(x, w, out, M, N, K, residual=res, ldx=ld, ldr=ld, ldc=ld, **kw)
    st.sync()
    assert torch.equal(out, apart)
    kept[:, K + N:K + 2 * N] = apart
    assert torch.equal(buf, kept)
