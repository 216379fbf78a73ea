"""The linear layers with their epilogue, dense and grouped by expert, against float64.

The operands hold small integers, so every product and every partial sum is exact in fp32 (and
in int32) whatever the order of the additions: |sum| <= 9 * K < 2^24.  What is left to err,
and what the tolerance counts, is (u = 2^-24, the half step of fp32):
  z      int8: two roundings, 2 u |z|; bf16 operands: none
  z + b  one rounding, u |z + b|
  act    its slope is at most 1.13 (taken as 1.2), and its own evaluation: __expf errs by
         2 + 1.17 |v| ulp, the quotient and 1 + e by a few more, (8 + 1.2 |v|) 2 u |act|; erff
         and tanhf by 2 ulp of values near one, |v| 2^-21 with the argument's roundings
  gate   the product's rounding, u, and each factor's error times the other
  + r    one rounding, u |y|
  out    half a step of the output type: 2^-8 (bf16) or 2^-24 (fp32) relative
"""
import numpy as np
import pytest

import qgemm

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ACTS = ["none", "relu", "gelu", "gelu_tanh", "silu"]
CANARY = -77.25


def act64(name, v):
    if name == "relu":
        return torch.clamp_min(v, 0)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / 2 ** 0.5)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3))
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def ints(g, shape, dtype, lo=-3, hi=4):
    return torch.randint(lo, hi, shape, generator=g, device="cuda").to(dtype)


class Case:
    """Inputs of one call; `offsets` (a list) makes it an expert call."""

    def __init__(self, kind, M, N, K, *, act="none", gated=False, bias=False, residual=False,
                 out="bf16", offsets=None, ldx=None, ldc=None, ldr=None, seed=0, shift=0):
        g = torch.Generator("cuda").manual_seed(seed + 1000 * M + 10 * N + K)
        self.kind, self.M, self.N, self.K = kind, M, N, K
        self.act, self.gated, self.offsets = act, gated, offsets
        E = 1 if offsets is None else len(offsets) - 1
        self.E = E
        nw = 2 * N if gated else N
        t = torch.bfloat16 if kind == "bf16" else torch.int8
        self.ldx, self.ldc = ldx or K, ldc or N
        self.ldr = ldr or N
        self.odt = torch.bfloat16 if out == "bf16" else torch.float32
        self.out_code = qgemm.BF16 if out == "bf16" else qgemm.F32
        # `shift` elements into a larger buffer: misaligned operands
        self.x = self._place(ints(g, (M, K), t), self.ldx, shift)
        self.w = self._place(ints(g, (E * nw, K), t), K, shift)
        scale = 1.0 / max(1.0, K ** 0.5)
        self.sx = (torch.rand(M, generator=g, device="cuda") + 0.5) * scale if kind == "w8a8" else None
        self.sw = torch.rand((E, nw), generator=g, device="cuda") + 0.5 if kind == "w8a8" else None
        self.bias = torch.randn((E, nw), generator=g, device="cuda") if bias else None
        self.residual = (self._place(torch.randn((M, N), generator=g, device="cuda").to(self.odt), self.ldr, 0)
                         if residual else None)
        self.buf = torch.full((M * self.ldc + 64,), CANARY, dtype=self.odt, device="cuda")
        self.out = torch.as_strided(self.buf, (M, N), (self.ldc, 1), 32)

    @staticmethod
    def _place(v, ld, shift):
        rows, width = v.shape
        buf = torch.zeros(max(1, rows * ld) + 16 + shift, dtype=v.dtype, device="cuda")
        view = torch.as_strided(buf, (rows, width), (ld, 1), shift)
        view.copy_(v)
        return view

    def call(self, ops, algo=qgemm.ALGO_AUTO, out=None):
        out = self.out if out is None else out
        kw = dict(bias=self.bias, act=ACTS.index(self.act), gated=self.gated,
                  out_dtype=self.out_code, ldc=self.ldc, algo=algo)
        if self.offsets is not None:
            off = torch.tensor(self.offsets, dtype=torch.int32, device="cuda")
            torch.cuda.synchronize()
            self._off = off
            if self.kind == "bf16":
                ops.expertLinearBf16NK(self.x, self.w, off, out, self.E, self.M, self.N, self.K,
                                       ldx=self.ldx, **kw)
            else:
                ops.w8a8ExpertLinear(self.x, self.w, self.sx, self.sw, off, out, self.E, self.M,
                                     self.N, self.K, lda=self.ldx, **kw)
            return
        kw.update(residual=self.residual, ldr=self.ldr)
        torch.cuda.synchronize()
        if self.kind == "bf16":
            ops.linearBf16NK(self.x, self.w, out, self.M, self.N, self.K, ldx=self.ldx, **kw)
        else:
            ops.w8a8Linear(self.x, self.w, self.sx, self.sw, out, self.M, self.N, self.K,
                           lda=self.ldx, **kw)

    def exact(self):
        """(value, tolerance, rows that are written)."""
        nw = self.w.shape[0] // self.E
        off = [0, self.M] if self.offsets is None else self.offsets
        y = torch.full((self.M, self.N), float("nan"), dtype=torch.float64, device="cuda")
        tol = torch.zeros_like(y)
        written = torch.zeros(self.M, dtype=torch.bool, device="cuda")
        uo = 2.0 ** -8 if self.odt == torch.bfloat16 else U
        for e in range(self.E):
            r0, r1 = off[e], off[e + 1]
            if not 0 <= r0 < r1 <= self.M:
                continue
            z = self.x[r0:r1].double() @ self.w[e * nw:(e + 1) * nw].double().t()
            ez = torch.zeros_like(z)
            if self.kind == "w8a8":
                z = z * self.sw[e].double() * self.sx[r0:r1].double()[:, None]
                ez = 2 * U * z.abs()
            if self.bias is not None:
                z = z + self.bias[e].double()
                ez = ez + U * z.abs()

            def activated(v, ev):
                a = act64(self.act, v)
                if self.act in ("none", "relu"):
                    return a, ev
                return a, 1.2 * ev + 2 * U * (8 + 1.2 * v.abs()) * a.abs() + 2.0 ** -21 * v.abs()

            if self.gated:
                a, ea = activated(z[:, :self.N], ez[:, :self.N])
                up, eu = z[:, self.N:], ez[:, self.N:]
                v = a * up
                ev = ea * up.abs() + a.abs() * eu + ea * eu + U * v.abs()
            else:
                v, ev = activated(z, ez)
            if self.residual is not None:
                v = v + self.residual[r0:r1].double()
                ev = ev + U * v.abs()
            y[r0:r1] = v
            tol[r0:r1] = ev + uo * (v.abs() + ev)
            written[r0:r1] = True
        return y, tol, written

    def check(self):
        y, tol, written = self.exact()
        got = self.out.double()
        w = written
        d = (got[w] - y[w]).abs()
        assert not torch.isnan(got[w]).any()
        over = d > tol[w]
        assert not over.any(), (f"{int(over.sum())} of {over.numel()} outside; worst "
                                f"{float((d / tol[w].clamp_min(1e-300)).max()):.3g} of the tolerance")
        # rows of no group and everything between the rows stay as they were
        assert (self.out[~w] == CANARY).all()
        mask = torch.ones(self.buf.numel(), dtype=torch.bool, device="cuda")
        torch.as_strided(mask, (self.M, self.N), (self.ldc, 1), 32).fill_(False)
        assert (self.buf[mask] == CANARY).all()


def run(gpu, case, algo=qgemm.ALGO_AUTO):
    _, st, ops = gpu
    case.call(ops, algo)
    st.sync()
    case.check()


SHAPES = [  # rows, features, K (multiples of 16 bytes in both types)
    (1, 128, 128), (1, 4096, 4096), (2, 17, 64), (3, 1000, 272), (15, 130, 1040), (16, 64, 16),
    (17, 200, 400), (32, 256, 4096), (33, 1001, 512), (64, 520, 656), (65, 96, 2048),
    (100, 2050, 128), (128, 384, 1536), (129, 300, 512), (200, 257, 4112), (256, 256, 64),
    (257, 520, 1040), (300, 1000, 208), (513, 264, 96), (1000, 777, 352), (2048, 2304, 256),
]


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_linear_shapes(gpu, kind, i):
    M, N, K = SHAPES[i]
    run(gpu, Case(kind, M, N, K, act=ACTS[i % 5], gated=i % 3 == 1, bias=i % 2 == 0,
                  residual=i % 4 < 2, out="f32" if i % 5 < 2 else "bf16"), qgemm.ALGO_TCGEN05)


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M", [5, 300])
def test_linear_epilogues(gpu, kind, act, gated, M):
    for bias, residual, out in ((True, True, "bf16"), (False, True, "f32"), (True, False, "f32"),
                                (False, False, "bf16")):
        run(gpu, Case(kind, M, 328, 512, act=act, gated=gated, bias=bias, residual=residual, out=out),
            qgemm.ALGO_TCGEN05)


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M,N,K", [(1, 7, 13), (3, 33, 1), (70, 65, 100), (40, 40, 0), (300, 48, 31)])
@pytest.mark.parametrize("gated", [False, True])
def test_linear_odd_k_runs_on_cuda_cores(gpu, kind, M, N, K, gated):
    run(gpu, Case(kind, M, N, K, act="silu", gated=gated, bias=True, residual=True, ldx=K + 3))
    if K % 16:
        with pytest.raises(qgemm.QGemmError) as e:
            Case(kind, M, N, K).call(gpu[2], qgemm.ALGO_TCGEN05)
        assert e.value.status == qgemm._lib.ERR_UNSUPPORTED


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_linear_strides_and_alignment(gpu, kind, M):
    # row pitches of the operands and of the outputs; pitches that rule the vector stores out
    run(gpu, Case(kind, M, 200, 256, bias=True, residual=True, ldx=256 + 32, ldc=208, ldr=216))
    run(gpu, Case(kind, M, 200, 256, residual=True, ldx=256 + 32, ldc=203, ldr=201, out="f32"))
    run(gpu, Case(kind, M, 203, 256, gated=True, act="gelu", bias=True))
    # operands that start off a 16-byte boundary, rows too: the CUDA-core path
    run(gpu, Case(kind, M, 40, 64, shift=1, bias=True))
    run(gpu, Case(kind, M, 40, 64, ldx=67, bias=True))


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M", [1, 64, 513])
@pytest.mark.parametrize("gated", [False, True])
def test_simt_agrees_with_tensor_cores(gpu, kind, M, gated):
    """The exact sums make every fp32 step the same on both paths, but for the gate's and the
    activation's contraction choices: both within the tolerance of the definition."""
    for algo in (qgemm.ALGO_SIMT, qgemm.ALGO_TCGEN05):
        run(gpu, Case(kind, M, 136, 192, act="silu", gated=gated, bias=True, residual=True), algo)


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M", [3, 400])
def test_linear_adds_onto_the_residual_in_place(gpu, kind, M):
    _, st, ops = gpu
    c = Case(kind, M, 264, 320, act="gelu", bias=True, residual=True)
    c.residual = c.out
    c.out.copy_(torch.randn(M, 264, device="cuda"))
    y, tol, _ = c.exact()
    c.call(ops)
    st.sync()
    assert ((c.out.double() - y).abs() <= tol).all()


def test_linear_rows_do_not_touch_each_other(gpu):
    """A row of NaN or infinities stays a row of them: other rows keep their bits (the tile's
    padding and its neighbours are columns of the same products)."""
    _, st, ops = gpu
    for M in (7, 300):
        a = Case("bf16", M, 264, 256, act="gelu", bias=True, out="f32")
        a.call(ops)
        st.sync()
        clean = a.out.clone()
        a.x[3] = float("nan")
        a.x[M - 1] = float("inf")
        a.call(ops)
        st.sync()
        keep = torch.ones(M, dtype=torch.bool, device="cuda")
        keep[3] = keep[M - 1] = False
        assert torch.equal(a.out[keep], clean[keep])
        assert torch.isnan(a.out[3]).all()


def test_activation_extremes(gpu):
    """Values far out on both sides, through the bias (K = 16 zeros): no NaN appears, the
    limits are kept."""
    _, st, ops = gpu
    v = torch.tensor([-3e38, -1e30, -1e4, -100., -88.5, -60., -20., -1e-30, 0., 1e-30, 20., 60.,
                      88.5, 100., 1e4, 1e18], device="cuda")
    x = torch.zeros(2, 16, dtype=torch.bfloat16, device="cuda")
    w = torch.zeros(16, 16, dtype=torch.bfloat16, device="cuda")
    out = torch.empty(2, 16, device="cuda")
    for act in ACTS:
        torch.cuda.synchronize()
        ops.linearBf16NK(x, w, out, 2, 16, 16, bias=v, act=ACTS.index(act), out_dtype=qgemm.F32)
        st.sync()
        ref = act64(act, v.double())
        if act == "gelu_tanh":  # the cube overflows past 1e12 in fp32: its limit is the value's
            ref = torch.where(v.abs() > 1e3, torch.clamp_min(v, 0).double(), ref)
        tol = 2.0 ** -20 * v.double().abs() + (8 + 1.2 * v.double().abs().clamp_max(90)) * 2 ** -22 * ref.abs()
        tol = torch.where(v < -20, torch.full_like(tol, 1e-6), tol)
        for row in out:
            assert not torch.isnan(row).any(), act
            assert ((row.double() - ref).abs() <= tol).all(), act


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
def test_far_rows_need_64_bit_offsets(gpu, kind):
    """Output rows 2^30 elements apart: the last row starts 2^31 elements in."""
    _, st, ops = gpu
    M, N, K, ldc = 3, 40, 64, 1 << 30
    c = Case(kind, M, N, K, bias=True, act="relu")
    c.buf = None
    big = torch.empty(2 * ldc + N, dtype=torch.bfloat16, device="cuda")
    c.ldc = ldc
    c.out = torch.as_strided(big, (M, N), (ldc, 1))
    for algo in (qgemm.ALGO_TCGEN05, qgemm.ALGO_SIMT):
        c.out.fill_(CANARY)
        c.call(ops, algo)
        st.sync()
        y, tol, _ = c.exact()
        assert ((c.out.double() - y).abs() <= tol).all()


# ---- grouped by expert ---------------------------------------------------------------------

OFFSETS = [
    [0, 5],                                     # one expert
    [0, 0, 1, 1],                               # one row among three experts
    [0, 3, 3, 20, 21, 40],                      # ragged, one empty, rows behind the last
    [2, 2, 9, 33, 70],                          # rows before the first belong to none
    [0, 100, 100, 100, 101],
    [0, 129, 258, 300],
    [0, 1, 300, 301, 600, 601, 900, 902],
    [0, 700, 700, 713, 1000],
    [0] * 30 + [64] + [64] * 33,                # 63 experts, one has all rows
]


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("i", range(len(OFFSETS)))
@pytest.mark.parametrize("gated", [False, True])
def test_expert_linear(gpu, kind, i, gated):
    off = OFFSETS[i]
    M = off[-1] + (6 if i % 2 == 0 else 0)
    run(gpu, Case(kind, M, 200 if i % 2 else 131, 272, act=ACTS[(i + gated) % 5], gated=gated,
                  bias=i % 3 != 0, out="f32" if i % 2 else "bf16", offsets=off),
        qgemm.ALGO_TCGEN05)


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
def test_expert_linear_no_rows_at_all(gpu, kind):
    run(gpu, Case(kind, 4, 64, 64, offsets=[0, 0, 0, 0]))
    run(gpu, Case(kind, 4, 64, 61, offsets=[0, 0, 0, 0]))


@pytest.mark.parametrize("kind,K", [("bf16", 264), ("w8a8", 272), ("bf16", 21), ("w8a8", 21)])
def test_expert_linear_1024_experts(gpu, kind, K):
    rng = np.random.default_rng(4)
    off = np.concatenate([[0], np.cumsum(rng.integers(0, 3, 1024))]).tolist()
    run(gpu, Case(kind, off[-1], 72, K, act="silu", gated=True, bias=True, offsets=off))


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
def test_expert_linear_many_rows_per_expert(gpu, kind):
    rng = np.random.default_rng(5)
    off = np.concatenate([[0], np.cumsum(rng.integers(200, 900, 7))]).tolist()
    run(gpu, Case(kind, off[-1], 520, 512, act="gelu", bias=True, offsets=off, ldc=528, ldx=528))


@pytest.mark.parametrize("algo", [qgemm.ALGO_TCGEN05, qgemm.ALGO_SIMT])
@pytest.mark.parametrize("M", [40, 400])
def test_bad_offsets_name_no_rows_and_are_reported(gpu, algo, M):
    """Offsets past M, negative or falling: that expert is skipped, the others are right, and
    the next sync says so, once."""
    _, st, ops = gpu
    for off in ([0, 10, 12, 20, 5], [-3, 4, 9, 9, 20], [0, 8, 8, M + 1, M + 2],
                [0, 2 ** 31 - 1, 2 ** 31 - 1, 4, 20]):
        c = Case("bf16", M, 72, 64, bias=True, offsets=off)
        c.call(ops, algo)
        with pytest.raises(qgemm.QGemmError) as e:
            st.sync()
        assert e.value.status == qgemm._lib.ERR_INVALID_ARG
        st.sync()
        c.check()


# ---- how calls live together ---------------------------------------------------------------

@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M", [1, 300])
def test_same_call_same_bits(gpu, kind, M):
    _, st, ops = gpu
    c = Case(kind, M, 1000, 4096, act="silu", gated=True, out="f32")
    if kind == "bf16":  # sums that do round, so that an order could show
        c.x.copy_(torch.randn_like(c.x.float()))
        c.w.copy_(torch.randn_like(c.w.float()))
    other = Case("w8a8", 50, 512, 512, bias=True)
    c.call(ops)
    st.sync()
    first = c.out.clone()
    for _ in range(5):
        other.call(ops)
        c.out.fill_(CANARY)
        c.call(ops)
        st.sync()
        assert torch.equal(c.out, first)


def test_two_streams_at_once(gpu):
    dev, _, _ = gpu
    cases = [Case("bf16", 1, 2048, 2048, bias=True), Case("w8a8", 300, 1024, 1024, act="gelu"),
             Case("w8a8", 20, 520, 2048, offsets=[0, 3, 9, 20]), Case("bf16", 257, 640, 512)]
    streams = [dev.stream() for _ in cases]
    try:
        for _ in range(20):
            for c, s in zip(cases, streams):
                c.call(qgemm.QuantizedGemmOps(s))
        for c, s in zip(cases, streams):
            s.sync()
            c.check()
    finally:
        for s in streams:
            s.destroy()


def test_captured_and_replayed(gpu):
    """Two graphs of the same calls, replayed in turn and on new inputs; the counts of the
    experts change between replays without a new capture."""
    dev, _, _ = gpu
    E, M, N, K = 4, 40, 264, 512
    c = Case("w8a8", M, N, K, act="silu", gated=True, offsets=[0, 10, 10, 25, 40])
    d = Case("bf16", 2, 520, 1024, act="gelu", bias=True, residual=True)
    off = torch.tensor(c.offsets, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    graphs = []
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        st = dev.wrap_stream(side.cuda_stream)
        ops = qgemm.QuantizedGemmOps(st)
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                ops.w8a8ExpertLinear(c.x, c.w, c.sx, c.sw, off, c.out, E, M, N, K,
                                     act=qgemm.ACT_SILU, gated=True)
                ops.linearBf16NK(d.x, d.w, d.out, 2, 520, 1024, bias=d.bias, residual=d.residual,
                                 act=qgemm.ACT_GELU)
            graphs.append(g)
    for i, new in enumerate(([0, 10, 10, 25, 40], [0, 0, 39, 40, 40], [0, 1, 2, 3, 4], [0, 40, 40, 40, 40])):
        c.offsets = new
        off.copy_(torch.tensor(new, dtype=torch.int32))
        c.out.fill_(CANARY)
        d.x.copy_(ints(torch.Generator("cuda").manual_seed(i), d.x.shape, torch.bfloat16))
        d.out.fill_(CANARY)
        torch.cuda.synchronize()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        c.check()
        d.check()
    del graphs
    st.destroy()


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M", [1, 33])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("N", [17, 1500, 2501, 4800, 11008, 20002])
def test_linear_few_rows_many_widths(gpu, kind, M, gated, N):
    """Few rows: the weight rows a tile and the cut of K follow the width."""
    run(gpu, Case(kind, M, N, 1040, act="silu", gated=gated, bias=True, residual=True),
        qgemm.ALGO_TCGEN05)


@pytest.mark.parametrize("avg", [20, 40, 94, 130])
@pytest.mark.parametrize("gated", [False, True])
def test_expert_linear_fp32_long_sums(gpu, avg, gated):
    """fp32 outputs of more than 512 values a sum, over ragged groups around the kernels' token
    tiles."""
    rng = np.random.default_rng(avg)
    off = np.concatenate([[0], np.cumsum(rng.integers(0, 2 * avg, 40))]).tolist()
    run(gpu, Case("bf16", off[-1], 392, 1304, act="gelu_tanh", gated=gated, bias=True, out="f32",
                  offsets=off))


@pytest.mark.parametrize("M", [1, 63, 65, 81, 97, 200, 300])
def test_linear_fp32_sums_keep_their_precision(gpu, M):
    """Random bf16 operands, K = 8192, fp32 out: sums in pieces of 512 values.  A piece loses up
    to one unit of the accumulator (2^-23 of the running sum, rounded toward zero) for each of
    its 512 / 16 MMAs; the running sum never passes sum |x w|, so the error stays below
    (32 + 16) 2^-23 of it (32 truncations a piece, 16 additions of pieces)."""
    _, st, ops = gpu
    N, K = 136, 8192
    g = torch.Generator("cuda").manual_seed(M)
    x = torch.randn(M, K, generator=g, device="cuda").bfloat16()
    w = torch.randn(N, K, generator=g, device="cuda").bfloat16()
    out = torch.empty(M, N, device="cuda")
    torch.cuda.synchronize()
    ops.linearBf16NK(x, w, out, M, N, K, out_dtype=qgemm.F32)
    st.sync()
    exact = x.double() @ w.double().t()
    bound = 48 * 2.0 ** -23 * (x.double().abs() @ w.double().abs().t())
    d = (out.double() - exact).abs()
    assert (d <= bound).all()
    # and in the mean far below what one accumulator over all of K loses (9e-6 of the result)
    assert float(d.norm() / exact.norm()) < 2e-6


@pytest.mark.parametrize("kind", ["bf16", "w8a8"])
@pytest.mark.parametrize("M,K,out", [(6, 4096, "bf16"), (2000, 512, "bf16"), (2000, 2048, "f32")])
def test_expert_linear_every_expert_empty(gpu, kind, M, K, out):
    """No tile at all, in each kernel: nothing is written and nothing waits."""
    run(gpu, Case(kind, M, 264, K, offsets=[0, 0, 0], out=out))
    run(gpu, Case(kind, M, 264, K, offsets=[M, M, M], out=out))


def test_linear_sizes_drawn(gpu):
    """Sizes drawn over their logarithm, with every epilogue: the kernels and cuts that the
    time model picks between."""
    rng = np.random.default_rng(2024)

    def log(lo, hi):
        return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))

    for i in range(120):
        kind = "bf16" if rng.random() < 0.5 else "w8a8"
        M, N, K = log(1, 900), log(8, 3000), log(1, 150) * 16
        off = None
        if rng.random() < 0.4:
            E = int(rng.choice([1, 2, 7, 40]))
            cuts = np.sort(rng.integers(0, M + 1, E + 1))
            off = cuts.tolist()
        run(gpu, Case(kind, M, N, K, act=ACTS[i % 5], gated=bool(rng.random() < 0.5),
                      bias=bool(rng.random() < 0.5), residual=off is None and bool(rng.random() < 0.5),
                      out="f32" if rng.random() < 0.4 else "bf16", offsets=off, seed=i),
            qgemm.ALGO_TCGEN05)
