"""The feed-forward operators of libqgemm as workloads: linear layers with bias, activation,
gate and residual in their epilogue, the same grouped by expert over ragged row counts, and
the routing, dispatch and combine steps around the experts.

``listed()`` and ``draw()`` give cases, ``prepare`` the inputs a serving program holds before
the call, ``run`` one pass: the plain torch form in 32 bits, or libqgemm's calls when ``own``
is set.  ``exact`` evaluates the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
LARGEST_FLOPS = 2.0 * 8192 * 2 * 14336 * 4096   # of "experts w8a8 prefill", the largest case
LARGEST_BYTES = 1.0e9


# ---- cases -------------------------------------------------------------------------------

def listed():
    return [
        # one decoded token through an output projection with its bias, added to the stream
        {"name": "linear bf16 one token", "op": "linear", "type": "bf16", "M": 1, "N": 4096,
         "K": 4096, "act": "none", "gated": False, "bias": True, "residual": True, "out": "bf16"},
        # a decode batch of 33 sequences through gate+up of a quantised 11008-wide block
        {"name": "linear w8a8 decode gated", "op": "linear", "type": "w8a8", "M": 33, "N": 11008,
         "K": 4096, "act": "silu", "gated": True, "bias": False, "residual": False, "out": "bf16"},
        # a prompt of 4096 tokens through the down projection, bias and residual fused
        {"name": "linear bf16 prefill", "op": "linear", "type": "bf16", "M": 4096, "N": 4096,
         "K": 11008, "act": "gelu", "gated": False, "bias": True, "residual": True, "out": "bf16"},
        # 16 decoded tokens, two experts each, through the experts' gate+up weights
        {"name": "experts w8a8 decode", "op": "experts", "type": "w8a8", "E": 8, "R": 32,
         "N": 14336, "K": 4096, "act": "silu", "gated": True, "bias": False, "skew": 0.5,
         "out": "bf16"},
        # 4096 prompt tokens, two experts each, the same weights
        {"name": "experts w8a8 prefill", "op": "experts", "type": "w8a8", "E": 8, "R": 8192,
         "N": 14336, "K": 4096, "act": "silu", "gated": True, "bias": False, "skew": 0.5,
         "out": "bf16"},
        # many small experts with ragged rows (some empty), bias and gelu, fp32 out
        {"name": "experts bf16 ragged", "op": "experts", "type": "bf16", "E": 64, "R": 6001,
         "N": 1544, "K": 2048, "act": "gelu_tanh", "gated": False, "bias": True, "skew": 1.0,
         "out": "f32"},
        # routing of one decode step and of a long prompt
        {"name": "route decode", "op": "route", "T": 16, "E": 8, "k": 2, "type": "f32",
         "renormalize": True},
        {"name": "route prefill", "op": "route", "T": 16384, "E": 64, "k": 8, "type": "bf16",
         "renormalize": False},
        # rows to their experts: a decode batch copied, a prompt quantised on the way
        {"name": "dispatch decode", "op": "dispatch", "type": "bf16", "quantize": False, "T": 33,
         "E": 8, "k": 2, "K": 4096},
        {"name": "dispatch prefill", "op": "dispatch", "type": "bf16", "quantize": True,
         "T": 8192, "E": 8, "k": 2, "K": 4096},
        # the experts' rows back to their tokens, weighted, onto the residual stream
        {"name": "combine decode", "op": "combine", "type": "bf16", "T": 16, "E": 8, "k": 2,
         "N": 4096, "residual": True, "out": "bf16"},
        {"name": "combine prefill", "op": "combine", "type": "bf16", "T": 8192, "E": 64, "k": 8,
         "N": 4096, "residual": True, "out": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "experts", "experts", "route", "dispatch", "combine"])
    if op in ("linear", "experts"):
        typ = rng.choice(["bf16", "w8a8"])
        step = 8 if typ == "bf16" else 16
        c = {"op": op, "type": typ}
        if op == "linear":
            c["M"] = _log(rng, 1, 8192)
        else:
            c["E"] = rng.choice([2, 5, 8, 16, 64, 128])
            c["R"] = _log(rng, 1, 8192)
        c["N"] = _log(rng, 256, 14336)
        if rng.random() < 0.75:
            c["N"] = -(-c["N"] // 8) * 8
        c["K"] = -(-_log(rng, 256, 11008) // step) * step
        c["act"] = rng.choice(ACTS)
        c["gated"] = rng.random() < 0.4
        c["bias"] = rng.random() < 0.5
        if op == "linear":
            c["residual"] = rng.random() < 0.5
        else:
            c["skew"] = rng.choice([0.0, 0.5, 1.0])
        c["out"] = rng.choice(["bf16", "bf16", "f32"])
        while True:
            w = work(c)
            if (w["flops"] <= LARGEST_FLOPS and _weight_bytes(c) <= LARGEST_BYTES
                    and _padded_values(c) <= 2.0e9):
                return c
            if _weight_bytes(c) > LARGEST_BYTES:
                c["N"] = max(256, c["N"] // 2)
            else:
                key = "M" if op == "linear" else "R"
                c[key] = max(1, c[key] // 2)
    T = _log(rng, 1, 16384 if op == "route" else 8192)
    E = rng.choice([4, 8, 16, 60, 64, 128, 256])
    k = min(E, rng.choice([1, 2, 4, 6, 8]))
    if op == "route":
        return {"op": op, "T": T, "E": E, "k": k, "type": rng.choice(["f32", "bf16"]),
                "renormalize": rng.random() < 0.5}
    width = _log(rng, 256, 8192)
    if rng.random() < 0.75:
        width = -(-width // 16) * 16
    while T * k * width > 8192 * 8 * 4096:
        T //= 2
    if op == "dispatch":
        return {"op": op, "type": rng.choice(["bf16", "f32"]), "quantize": rng.random() < 0.5,
                "T": T, "E": E, "k": k, "K": width}
    return {"op": op, "type": rng.choice(["bf16", "f32"]), "T": T, "E": E, "k": k, "N": width,
            "residual": rng.random() < 0.5, "out": rng.choice(["bf16", "f32"])}


# ---- the work a case cannot do without ---------------------------------------------------

def _rows_of_weights(c):
    return 2 * c["N"] if c["gated"] else c["N"]


def _size(t):
    return {"bf16": 2, "f32": 4, "w8a8": 1}[t]


def _weight_bytes(c):
    return c.get("E", 1) * _rows_of_weights(c) * c["K"] * _size(c["type"])


def _padded_values(c):
    """Values that the plain form of the experts' products holds, groups padded alike."""
    if c["op"] != "experts":
        return 0.0
    share = 1.0 / sum((i + 1.0) ** -c["skew"] for i in range(c["E"]))
    return c["E"] * c["R"] * share * (c["K"] + _rows_of_weights(c))


def work(case):
    c = case
    if c["op"] in ("linear", "experts"):
        e = _size(c["type"])
        M = c["M"] if c["op"] == "linear" else c["R"]
        groups = 1 if c["op"] == "linear" else min(c["E"], c["R"])
        nw = _rows_of_weights(c)
        b = M * c["K"] * e + groups * nw * c["K"] * e + M * c["N"] * _size(c["out"])
        if c["type"] == "w8a8":
            b += 4 * M + 4 * groups * nw
        if c["bias"]:
            b += 4 * groups * nw
        if c.get("residual"):
            b += M * c["N"] * _size(c["out"])
        if c["op"] == "experts":
            b += 4 * (c["E"] + 1)
        return {"bytes": float(b), "flops": 2.0 * M * nw * c["K"]}
    T, k = c["T"], c["k"]
    if c["op"] == "route":
        b = T * c["E"] * _size(c["type"]) + T * k * 12 + 4 * (c["E"] + 1)
        return {"bytes": float(b), "flops": 4.0 * T * c["E"]}
    if c["op"] == "dispatch":
        e = _size(c["type"])
        b = T * c["K"] * e + T * k * 4 + T * k * c["K"] * (1 if c["quantize"] else e)
        if c["quantize"]:
            b += 4 * T * k
        return {"bytes": float(b), "flops": 2.0 * T * c["K"]}
    e, o = _size(c["type"]), _size(c["out"])
    b = T * k * (c["N"] * e + 8) + T * c["N"] * o * (2 if c["residual"] else 1)
    return {"bytes": float(b), "flops": 2.0 * T * k * c["N"]}


# ---- inputs ------------------------------------------------------------------------------

def _dtype(t):
    return {"bf16": torch.bfloat16, "f32": torch.float32}[t]


def _uniform(g, shape, lo, hi):
    return torch.empty(shape, device=DEV).uniform_(lo, hi, generator=g)


def _normal(g, shape, std, dtype):
    return (torch.empty(shape, device=DEV).normal_(0.0, std, generator=g)).to(dtype)


def _int8(g, shape):
    return torch.empty(shape, device=DEV, dtype=torch.int8).random_(-127, 128, generator=g)


def _counts(case, seed):
    """Rows of every expert: a multinomial over popularities that fall off as 1 / rank^skew."""
    g = torch.Generator().manual_seed(seed * 2 + 1)
    E, R = case["E"], case["R"]
    p = torch.arange(1, E + 1, dtype=torch.float64).pow(-case["skew"])[torch.randperm(E, generator=g)]
    ids = torch.multinomial(p / p.sum(), R, replacement=True, generator=g)
    return torch.bincount(ids, minlength=E)


def _pairs(case, g):
    """Routing of T tokens as the routing operator leaves it: expert ids, rows, weights."""
    T, E, k = case["T"], case["E"], case["k"]
    ids = torch.rand((T, E), device=DEV, generator=g).topk(k, dim=1).indices
    order = torch.argsort(ids.reshape(-1), stable=True)
    rows = torch.empty(T * k, dtype=torch.int32, device=DEV)
    rows[order] = torch.arange(T * k, dtype=torch.int32, device=DEV)
    w = torch.softmax(torch.randn((T, k), device=DEV, generator=g), dim=1)
    return rows.reshape(T, k), w


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    c, s = case, {"case": case}
    if c["op"] in ("linear", "experts"):
        M = c["M"] if c["op"] == "linear" else c["R"]
        E, nw, K = c.get("E", 1), _rows_of_weights(c), c["K"]
        wshape = (nw, K) if c["op"] == "linear" else (E, nw, K)
        # activations ~ N(0, 1); weights and scales so that the products are of order one
        if c["type"] == "bf16":
            s["x"] = _normal(g, (M, K), 1.0, torch.bfloat16)
            s["w"] = _normal(g, wshape, K ** -0.5, torch.bfloat16)
        else:
            s["x"], s["w"] = _int8(g, (M, K)), _int8(g, wshape)
            s["sx"] = _uniform(g, (M,), 0.01, 0.03)
            s["sw"] = _uniform(g, wshape[:-1], 0.5, 1.5) / (73.0 * 73.0 * 0.02 * K ** 0.5)
        s["bias"] = _normal(g, wshape[:-1], 0.5, torch.float32) if c["bias"] else None
        s["residual"] = _normal(g, (M, c["N"]), 1.0, _dtype(c["out"])) if c.get("residual") else None
        s["out"] = torch.empty((M, c["N"]), dtype=_dtype(c["out"]), device=DEV)
        if c["op"] == "experts":
            n = _counts(c, seed)
            off = torch.zeros(E + 1, dtype=torch.int64)
            off[1:] = torch.cumsum(n, 0)
            s["offsets"] = off.to(torch.int32).to(DEV)
            s["most"] = int(n.max())   # the largest group, for the padded plain form
        return s
    if c["op"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        s["logits"] = _normal(g, (T, E), 1.5, _dtype(c["type"]))
        s["weights"] = torch.empty((T, k), device=DEV)
        s["experts"] = torch.empty((T, k), dtype=torch.int32, device=DEV)
        s["offsets"] = torch.empty(E + 1, dtype=torch.int32, device=DEV)
        s["rows"] = torch.empty((T, k), dtype=torch.int32, device=DEV)
        return s
    T, k = c["T"], c["k"]
    s["rows"], s["weights"] = _pairs(c, g)
    if c["op"] == "dispatch":
        s["x"] = _normal(g, (T, c["K"]), 1.0, _dtype(c["type"]))
        if c["quantize"]:
            s["q"] = torch.empty((T * k, c["K"]), dtype=torch.int8, device=DEV)
            s["sq"] = torch.empty(T * k, device=DEV)
        else:
            s["out"] = torch.empty((T * k, c["K"]), dtype=_dtype(c["type"]), device=DEV)
        return s
    s["y"] = _normal(g, (T * k, c["N"]), 1.0, _dtype(c["type"]))
    s["residual"] = _normal(g, (T, c["N"]), 1.0, _dtype(c["out"])) if c["residual"] else None
    s["out"] = torch.empty((T, c["N"]), dtype=_dtype(c["out"]), device=DEV)
    return s


# ---- the plain forms ---------------------------------------------------------------------

def _act(name, v):
    if name == "relu":
        return torch.maximum(v, torch.zeros((), device=v.device))
    if name == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * 0.7071067811865476))
    if name == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _finish(c, z):
    """Activation, or activated gate times up, of the biased products."""
    if not c["gated"]:
        return _act(c["act"], z)
    N = c["N"]
    return _act(c["act"], z[..., :N]) * z[..., N:]


def _plain_linear(s):
    c = s["case"]
    z = torch.matmul(s["x"].float(), s["w"].float().t())
    if c["type"] == "w8a8":
        z = z * s["sw"] * s["sx"][:, None]
    if s["bias"] is not None:
        z = z + s["bias"]
    y = _finish(c, z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out"].dtype)


def _plain_experts(s):
    """Every group padded to the largest, one batched product, the real rows taken back."""
    c = s["case"]
    R, E, cap = c["R"], c["E"], s["most"]
    off = s["offsets"].long()
    p = torch.arange(R, device=DEV)
    e = torch.searchsorted(off, p, right=True) - 1
    slot = e * cap + (p - off[e])
    x = torch.zeros((E * cap, c["K"]), device=DEV)
    x[slot] = s["x"].float()
    z = torch.bmm(x.view(E, cap, c["K"]), s["w"].float().transpose(1, 2))
    z = z.reshape(E * cap, -1)[slot]
    if c["type"] == "w8a8":
        z = z * s["sw"][e] * s["sx"][:, None]
    if s["bias"] is not None:
        z = z + s["bias"][e]
    return _finish(c, z).to(s["out"].dtype)


def _plain_route(s):
    c = s["case"]
    T, E, k = c["T"], c["E"], c["k"]
    v = s["logits"].float()
    # largest first, ties to the lowest index: a stable descending sort
    experts = torch.sort(v, dim=1, descending=True, stable=True).indices[:, :k]
    p = torch.exp(v - v.max(dim=1, keepdim=True).values)
    chosen = p.gather(1, experts)
    total = chosen.sum(1, keepdim=True) if c["renormalize"] else p.sum(1, keepdim=True)
    flat = experts.reshape(-1)
    order = torch.sort(flat, stable=True).indices
    rows = torch.empty_like(flat, dtype=torch.int32)
    rows[order] = torch.arange(T * k, dtype=torch.int32, device=DEV)
    n = torch.zeros(E, dtype=torch.int64, device=DEV).index_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64, device=DEV), torch.cumsum(n, 0)])
    return {"weights": chosen / total, "experts": experts.to(torch.int32),
            "offsets": offsets.to(torch.int32), "rows": rows.reshape(T, k)}


def _plain_dispatch(s):
    c = s["case"]
    T, k, K = c["T"], c["k"], c["K"]
    rows = s["rows"].long().reshape(-1)
    x = s["x"]
    if not c["quantize"]:
        out = torch.empty((T * k, K), dtype=x.dtype, device=DEV)
        out[rows] = x[:, None, :].expand(T, k, K).reshape(T * k, K)
        return {"out": out}
    f = x.float()
    most = f.abs().amax(1)
    full = torch.full_like(most, 127.0)
    mul = torch.where(most > 1e-6, full / most, torch.ones_like(most))
    q = torch.clamp(torch.trunc(f * mul[:, None]), -128, 127).to(torch.int8)
    scale = most / full
    qs = torch.empty((T * k, K), dtype=torch.int8, device=DEV)
    sq = torch.empty(T * k, device=DEV)
    qs[rows] = q[:, None, :].expand(T, k, K).reshape(T * k, K)
    sq[rows] = scale[:, None].expand(T, k).reshape(-1)
    return {"values": qs * sq[:, None], "scales": sq}


def _plain_combine(s):
    c = s["case"]
    y = s["y"][s["rows"].long()].float()
    out = (s["weights"][:, :, None] * y).sum(1)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(s["out"].dtype)


_PLAIN = {"linear": _plain_linear, "experts": _plain_experts, "route": _plain_route,
          "dispatch": _plain_dispatch, "combine": _plain_combine}


# ---- libqgemm's calls ---------------------------------------------------------------------

_handles = {}


def _ops():
    """The library on the current device and stream; a program opens them once and keeps them.
    (Asked for as torch's compiled code does: 0.2 us, where the Python object of
    torch.cuda.current_stream() takes 3.)"""
    device = torch._C._cuda_getDevice()
    stream = torch._C._cuda_getCurrentRawStream(device)
    ops = _handles.get((device, stream))
    if ops is None:
        import os
        import sys
        package = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                               "cuda-triton-scala_b200")
        if package not in sys.path:
            sys.path.insert(0, package)
        import qgemm
        if device not in _handles:
            _handles[device] = qgemm.Device(device)
        lib = qgemm.QuantizedGemmOps(_handles[device].wrap_stream(stream))
        acts = {"none": qgemm.ACT_NONE, "relu": qgemm.ACT_RELU, "gelu": qgemm.ACT_GELU,
                "gelu_tanh": qgemm.ACT_GELU_TANH, "silu": qgemm.ACT_SILU}
        ops = _handles[device, stream] = (lib, acts, {"bf16": qgemm.BF16, "f32": qgemm.F32})
    return ops


def _own(s):
    c = s["case"]
    ops, acts, types = _ops()
    op = c["op"]
    if op == "linear":
        M, N, K = c["M"], c["N"], c["K"]
        if c["type"] == "bf16":
            ops.linearBf16NK(s["x"], s["w"], s["out"], M, N, K, bias=s["bias"],
                             residual=s["residual"], act=acts[c["act"]], gated=c["gated"],
                             out_dtype=types[c["out"]])
        else:
            ops.w8a8Linear(s["x"], s["w"], s["sx"], s["sw"], s["out"], M, N, K, bias=s["bias"],
                           residual=s["residual"], act=acts[c["act"]], gated=c["gated"],
                           out_dtype=types[c["out"]])
        return s["out"]
    if op == "experts":
        E, R, N, K = c["E"], c["R"], c["N"], c["K"]
        if c["type"] == "bf16":
            ops.expertLinearBf16NK(s["x"], s["w"], s["offsets"], s["out"], E, R, N, K,
                                   bias=s["bias"], act=acts[c["act"]], gated=c["gated"],
                                   out_dtype=types[c["out"]])
        else:
            ops.w8a8ExpertLinear(s["x"], s["w"], s["sx"], s["sw"], s["offsets"], s["out"], E, R,
                                 N, K, bias=s["bias"], act=acts[c["act"]], gated=c["gated"],
                                 out_dtype=types[c["out"]])
        return s["out"]
    T, k = c["T"], c["k"]
    if op == "route":
        ops.routeTopK(s["logits"], s["weights"], s["experts"], s["offsets"], s["rows"], T, c["E"],
                      k, renormalize=c["renormalize"], in_dtype=types[c["type"]])
        return {n: s[n] for n in ("weights", "experts", "offsets", "rows")}
    if op == "dispatch":
        if c["quantize"]:
            ops.dispatchRowsQuantized(s["x"], s["rows"], s["q"], s["sq"], T, k, c["K"], T * k,
                                      in_dtype=types[c["type"]])
            return {"values": s["q"] * s["sq"][:, None], "scales": s["sq"]}
        ops.dispatchRows(s["x"], s["rows"], s["out"], T, k, c["K"], T * k,
                         dtype=types[c["type"]])
        return {"out": s["out"]}
    ops.combineRows(s["y"], s["rows"], s["weights"], s["out"], T, k, c["N"], T * k,
                    residual=s["residual"], in_dtype=types[c["type"]], out_dtype=types[c["out"]])
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits ------------------------------------------------------------

def _exact_act(name, v):
    if name == "relu":
        return torch.clamp_min(v, 0.0)
    if name == "gelu":
        return v * 0.5 * torch.special.erfc(-v / math.sqrt(2.0))
    if name == "gelu_tanh":
        u = math.sqrt(2.0 / math.pi) * (v + 0.044715 * v ** 3)
        return v * torch.sigmoid(2.0 * u)
    if name == "silu":
        return v * torch.sigmoid(v)
    return v


def _exact_rows(s, r0, r1, e):
    """Rows r0..r1 through the weights of expert e (None: the only weights there are)."""
    c, N = s["case"], s["case"]["N"]
    pick = (lambda t: t) if e is None else (lambda t: t[e])
    x = s["x"][r0:r1].double()
    y = torch.empty((r1 - r0, N), dtype=torch.float64, device=DEV)
    for n0 in range(0, N, 4096):
        n1 = min(N, n0 + 4096)

        def part(first):
            z = x @ pick(s["w"])[first + n0:first + n1].double().t()
            if c["type"] == "w8a8":
                z *= s["sx"][r0:r1].double()[:, None]
                z *= pick(s["sw"])[first + n0:first + n1].double()
            if s["bias"] is not None:
                z += pick(s["bias"])[first + n0:first + n1].double()
            return z

        y[:, n0:n1] = _exact_act(c["act"], part(0))
        if c["gated"]:
            y[:, n0:n1] *= part(N)
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "linear":
        y = _exact_rows(s, 0, c["M"], None)
        return y + s["residual"].double() if s["residual"] is not None else y
    if c["op"] == "experts":
        off = s["offsets"].tolist()
        y = torch.empty((c["R"], c["N"]), dtype=torch.float64, device=DEV)
        for e in range(c["E"]):
            if off[e + 1] > off[e]:
                y[off[e]:off[e + 1]] = _exact_rows(s, off[e], off[e + 1], e)
        return y
    T, k = c["T"], c["k"]
    if c["op"] == "route":
        v = s["logits"].double()
        top = v.topk(k, dim=1).values
        over = top if c["renormalize"] else v
        return {"weights": torch.exp(top - torch.logsumexp(over, 1, keepdim=True)),
                "experts": None, "offsets": None, "rows": None}
    rows = s["rows"].long()
    if c["op"] == "dispatch":
        if not c["quantize"]:
            out = torch.zeros((T * k, c["K"]), dtype=torch.float64, device=DEV)
            out[rows.reshape(-1)] = s["x"].double().repeat_interleave(k, 0)
            return {"out": out}
        sq = torch.zeros(T * k, dtype=torch.float64, device=DEV)
        sq[rows.reshape(-1)] = (s["x"].double().abs().amax(1) / 127.0).repeat_interleave(k, 0)
        # a value's step is decided by the 32-bit product that defines it
        return {"values": None, "scales": sq}
    out = torch.zeros((T, c["N"]), dtype=torch.float64, device=DEV)
    for j in range(k):
        out += s["weights"][:, j:j + 1].double() * s["y"][rows[:, j]].double()
    return out + s["residual"].double() if s["residual"] is not None else out
