"""Sizes past which the kernels' 32-bit counts could wrap: refused on the host.  Every check
answers before the device is touched; what passes them all fails on the null stream."""
import pytest

import qgemm._lib as L
from test_linear_args import CALLS, LINEARS, status

MOST = 1 << 30


@pytest.mark.parametrize("name", LINEARS)
@pytest.mark.parametrize("size", ["M", "N", "K"])
def test_linear_sizes_past_2_30_are_refused(name, size):
    """M, N or K above 2^30 (the loops step past the last element by up to a tile of 32, and
    row tiles are rounded up in int)."""
    pitch = {"M": {}, "N": {"ldc": MOST + 1}, "K": {("lda" if "w8a8" in name else "ldx"): MOST + 1}}[size]
    if size == "N" and "residual" in CALLS[name]:
        pitch["ldr"] = MOST + 1
    small = {"M": 1, "N": 1, "K": 1}
    small[size] = MOST + 1
    extra = {"E": 1} if "expert" in name else {}
    assert status(name, out=1 << 50, **pitch, **small, **extra) == L.ERR_UNSUPPORTED
    if size == "K" and "w8a8" in name:
        return  # int8 sums end at 131071
    small[size] = MOST
    far = {("A" if "w8a8" in name else "x"): 1 << 45, ("B" if "w8a8" in name else "w"): 1 << 46}
    assert status(name, out=1 << 50, **far, **pitch, **small, **extra) == L.ERR_BAD_HANDLE


@pytest.mark.parametrize("name,size", [("qgemm_route_topk", "T"), ("qgemm_dispatch_rows", "T"),
                                       ("qgemm_dispatch_rows", "K"),
                                       ("qgemm_dispatch_rows_quantized", "T"),
                                       ("qgemm_dispatch_rows_quantized", "K"),
                                       ("qgemm_combine_rows", "T"), ("qgemm_combine_rows", "N")])
def test_row_sizes_past_2_30_are_refused(name, size):
    """More than 2^30 tokens or values a row (a thread's index steps past the end by a block's
    width)."""
    small = {"T": 1, "k": 1}
    if name == "qgemm_route_topk":
        small["E"] = 1
        far = {"logits": 1 << 40, "weights": 1 << 41, "experts": 1 << 42, "offsets": 1 << 43, "rows": 1 << 44}
    else:
        small["R"] = 1
        small["N" if "combine" in name else "K"] = 1
        far = {"rows": 1 << 40}
        far.update({"y" if "combine" in name else "x": 1 << 41})
        far.update({"q" if "quantized" in name else "out": 1 << 42})
        if "quantized" in name:
            far["sA"] = 1 << 43
        if "combine" in name:
            far["weights"] = 1 << 44
    small[size] = MOST + 1
    assert status(name, **small, **far) == L.ERR_UNSUPPORTED
    small[size] = MOST
    assert status(name, **small, **far) == L.ERR_BAD_HANDLE
