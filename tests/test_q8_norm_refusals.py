"""Codes of csdr_add_rms_norm that would be written over what the call reads or over its other outputs: refused before
a launch, as csdr_q8_quantize's are."""
import pytest

from cortexsdr_amd import _lib

X, RESIDUAL, OUT, Y, CODES, SCALES, W = (4096 * i for i in range(1, 8))  # addresses that no refused call reads


@pytest.mark.parametrize("codes", [X, RESIDUAL, OUT, Y])
def test_codes_are_another(codes):
    lib = _lib.load()
    rc = lib.csdr_add_rms_norm(X, 0, 0, RESIDUAL, 0, 0, OUT, W, 1e-5, 2, 100, Y, codes, SCALES, None)
    assert rc == -1 and b"another output" in lib.csdr_last_error()


def test_codes_are_x_without_a_stream():
    lib = _lib.load()
    assert lib.csdr_add_rms_norm(X, 0, 0, None, 0, 0, None, W, 1e-5, 2, 100, None, X, SCALES, None) == -1
    assert b"another output" in lib.csdr_last_error()
