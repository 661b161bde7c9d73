"""Outputs that share a byte with the input are refused, by the rows' own bytes; without a GPU (the addresses are never read: every
call here is refused)."""
import pytest

from hecate_amd import _lib

A = 1 << 20
F32, BF16, F16 = 0, 1, 2


def refused(rc, word="overlap"):
    assert rc == 1 and word.encode() in _lib.lib().hmoe_last_error(), (rc, _lib.lib().hmoe_last_error())


@pytest.mark.parametrize("M", [1, 2, 7])
def test_rows_that_share_a_byte(M):
    """rows of 64 bf16 values, 96 apart (a row of 1: its own bytes alone)"""
    L = _lib.lib()
    pitch = 192

    def linear(y, ydt=BF16, N=8, ldy=96):
        return L.hmoe_i8_linear(A, BF16, 96, M, 8 * A, 64, 9 * A, N, 64, None, y, ydt, ldy, 10 * A, None)

    for y in (A, A + 126, A - 14, A + pitch * (M - 1) + 126, A + pitch * (M - 1)):
        refused(linear(y))
    refused(linear(A - 4 * 8 + 4, F32, 8, 48))
    refused(linear(A + 124, F32, 8, 48))
    refused(L.hmoe_i8_quantize(A, BF16, 96, M, 64, A + 112, 192, 5 * A, None))
    refused(L.hmoe_i8_quantize(A, BF16, 96, M, 64, A - 48, 192, 5 * A, None))
    refused(L.hmoe_i8_matmul(A, 192, 5 * A, M, 8 * A, 64, 9 * A, 8, 64, None, A + 60, F32, 48, None))
    if M > 1:
        # the next row's first byte, and from before the first row into it
        refused(linear(A + pitch - 14))
        refused(linear(A + 128, N=33))
        # other distances between the rows: by their whole spans
        refused(linear(A + 128, ldy=80))
