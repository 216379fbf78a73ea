"""ExpertMLP -- a mixture-of-experts feed-forward layer on W8A8 weights: the expert layers
together with the routing, dispatch and combine steps around them, over buffers made once."""
from __future__ import annotations

from . import _lib as L
from .runtime import Buffer


class ExpertMLP:
    """out[t] = residual[t] + sum_j p[t,j] * W2_e( act(W1gate_e x[t]) * (W1up_e x[t]) ), e the
    j-th expert of token t.

      router  bf16 [E, H]       logits = x router^T, fp32
      w1, s1  int8 [E, 2F, H], f32 [E, 2F]   gate rows, then up rows
      w2, s2  int8 [E, H, F],  f32 [E, H]

    Activations are quantised per token on the way into each product.  The object owns its
    intermediate buffers (for up to ``max_tokens`` tokens), so calls on one object must be
    ordered: one stream, or one object per stream (and per captured graph that may run beside
    another).  A call is seven launches (eight for many tokens), allocates nothing, waits for nothing on the host and
    can be captured into a CUDA graph after one call outside it.
    """

    def __init__(self, ops, router, w1, s1, w2, s2, *, E: int, k: int, H: int, F: int,
                 max_tokens: int, renormalize: bool = True, act: int = L.ACT_SILU):
        if not (1 <= k <= E) or H < 1 or F < 1 or max_tokens < 1:
            raise ValueError(f"bad ExpertMLP sizes E={E} k={k} H={H} F={F} max_tokens={max_tokens}")
        self.ops, self.E, self.k, self.H, self.F = ops, E, k, H, F
        self.max_tokens, self.renormalize, self.act = max_tokens, renormalize, act
        self.router, self.w1, self.s1, self.w2, self.s2 = router, w1, s1, w2, s2
        dev = ops.stream.dev
        T, R = max_tokens, max_tokens * k
        sizes = {"logits": 4 * T * E, "weights": 4 * R, "experts": 4 * R, "offsets": 4 * (E + 1),
                 "rows": 4 * R, "xq": R * H, "sx": 4 * R, "h": 2 * R * F, "hq": R * F,
                 "sh": 4 * R, "y": 2 * R * H}
        for name, nbytes in sizes.items():
            setattr(self, name, Buffer(dev, nbytes))

    def __call__(self, x, out, T: int, *, residual=None):
        """x, out, residual bf16 [T, H] (residual may be out)."""
        if not 0 <= T <= self.max_tokens:
            raise ValueError(f"{T} tokens; this layer holds {self.max_tokens}")
        if T == 0:
            return
        o, E, k, H, F, R = self.ops, self.E, self.k, self.H, self.F, T * self.k
        o.linearBf16NK(x, self.router, self.logits, T, E, H, out_dtype=L.F32)
        o.routeTopK(self.logits, self.weights, self.experts, self.offsets, self.rows, T, E, k,
                    renormalize=self.renormalize)
        o.dispatchRowsQuantized(x, self.rows, self.xq, self.sx, T, k, H, R)
        o.w8a8ExpertLinear(self.xq, self.w1, self.sx, self.s1, self.offsets, self.h, E, R, F, H,
                           act=self.act, gated=True)
        o.quantizePerToken(self.h, self.hq, self.sh, R, F)
        o.w8a8ExpertLinear(self.hq, self.w2, self.sh, self.s2, self.offsets, self.y, E, R, H, F)
        o.combineRows(self.y, self.rows, self.weights, out, T, k, H, R, residual=residual)

    def close(self):
        """Frees the buffers (after the work that uses them)."""
        for v in list(vars(self).values()):
            if isinstance(v, Buffer):
                v.free()
