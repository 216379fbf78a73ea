"""Which of a linear layer's buffers may lie where: outputs on any input are refused.  Every check answers before the device is touched;
what passes them all fails on the null stream."""
import pytest

import qgemm._lib as L
from test_linear_args import CALLS, LINEARS, big, status

OK = L.ERR_BAD_HANDLE


@pytest.mark.parametrize("name", LINEARS)
def test_out_on_any_input_is_refused(name):
    """8 rows of 32 bf16 features (64 bytes): out is [out, out + 512)."""
    out, bad = big(2), L.ERR_INVALID_ARG
    small = ["bias"] + (["sA", "sB"] if "w8a8" in name else []) + (["offsets"] if "expert" in name else [])
    for which in small:
        assert status(name, **{which: out}) == bad, which
        assert status(name, **{which: out + 508}) == bad, which
        assert status(name, **{which: out + 512}) == OK, which
    # an input that ends where out begins, and one that reaches into it
    length = {"bias": 32 * 4, "sA": 8 * 4, "sB": 32 * 4, "offsets": 5 * 4}
    for which in small:
        n = length[which] * (4 if "expert" in name and which in ("bias", "sB") else 1)
        assert status(name, **{which: out - n}) == OK, which
        assert status(name, **{which: out - n + 4}) == bad, which
