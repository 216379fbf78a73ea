"""Which of a linear layer's buffers may lie where: outputs on any input are refused, columns of
one wider buffer that share no byte are not.  Every check answers before the device is touched;
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
    # between the rows of an out with a wider pitch
    if "bias" in small and "expert" not in name:
        assert status(name, ldc=128, bias=out + 64) == OK
        assert status(name, ldc=128, bias=out + 64 + 68) == bad   # reaches the next row


@pytest.mark.parametrize("name", LINEARS)
def test_columns_of_one_buffer(name):
    """x and out, or out and the residual, side by side in rows of one buffer."""
    x, ld = ("A", "lda") if "w8a8" in name else ("x", "ldx")
    xb = 64 if "w8a8" in name else 128        # bytes of 64 values of a row of x
    pitch = {ld: 512 // (1 if "w8a8" in name else 2), "ldc": 256}     # both 512 bytes
    at = CALLS[name][x]
    assert status(name, **pitch, out=at + xb) == OK
    assert status(name, **pitch, out=at + 512 - 64) == OK
    assert status(name, **pitch, out=at + xb - 16) == L.ERR_INVALID_ARG
    assert status(name, **pitch, out=at + 512 - 48) == L.ERR_INVALID_ARG   # into the next row of x
    assert status(name, **pitch, out=at - 512 + xb) == OK                  # a row earlier
    # other pitches are compared as whole ranges
    assert status(name, **{**pitch, "ldc": 260}, out=at + xb) == L.ERR_INVALID_ARG
    if "residual" in CALLS[name]:
        out = big(2)
        assert status(name, ldc=256, ldr=256, residual=out + 64) == OK
        assert status(name, ldc=256, ldr=256, residual=out + 60) == L.ERR_INVALID_ARG
        assert status(name, ldc=256, ldr=256, residual=out) == OK
