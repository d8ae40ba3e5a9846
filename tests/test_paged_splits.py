"""How far csdr_paged_attn splits a sequence's positions, read off the workspace that a call asks
for, without a GPU: the refused calls end before a launch."""
import ctypes as C

import pytest

from cortexsdr_amd import _lib
from test_paged_refusals import OUT, WORKSPACE, P, kv


def refuses(n_bytes, tokens, **opt):
    """Whether a workspace of n_bytes is too small for a call of one long sequence."""
    rc = _lib.load().csdr_paged_attn(
        kv(n_seqs=1, table_stride=4096), P, 0, tokens, None, 0, 4, 0, 0, 0.0,
        C.byref(_lib.AttnOptions(**opt)), OUT, P, n_bytes, None)
    return rc == WORKSPACE


def bytes_of(tokens, splits):
    return tokens * 4 * splits * (8 + 64 * 4)


@pytest.mark.parametrize("tokens,unit", [(1, 128), (40, 512)])
@pytest.mark.parametrize("window", [1, 256])
def test_a_prefix_beside_a_window_is_split(tokens, unit, window):
    """A prefix may be long, whatever the window: at least as many splits as 4096 positions have."""
    assert refuses(bytes_of(tokens, 4096 // unit) - 1, tokens, window=window, prefix=P)


@pytest.mark.parametrize("tokens,window", [(1, 256), (40, 2048), (1, 0)])
def test_the_workspace_function_is_enough(tokens, window):
    """What csdr_paged_attn_workspace_bytes says is no less than any options need."""
    need = _lib.load().csdr_paged_attn_workspace_bytes(kv(n_seqs=1, table_stride=4096), tokens, None,
                                                       0, 4, 0)
    assert need >= bytes_of(tokens, 8)
    assert refuses(bytes_of(tokens, 2) - 1, tokens, window=window)


def test_page_bytes_of_more_heads_than_a_cache_has():
    """A shape that no call takes has no size."""
    f = _lib.load().csdr_paged_page_bytes
    assert f(1, 16, 65535, 64) > 0 and f(1, 16, 65536, 64) == 0 and f(2, 4096, 2 ** 31 - 1, 128) == 0


@pytest.mark.parametrize("heads", [65536, 98304])
def test_workspace_of_more_heads_than_a_call_has(heads):
    f = _lib.load().csdr_paged_attn_workspace_bytes
    wide = kv(n_kv_heads=32768)
    assert f(wide, 2, None, 0, heads, 0) == 0 and f(wide, 2, None, 0, 32768, 0) > 0


@pytest.mark.parametrize("dtype", [1, 2])
@pytest.mark.parametrize("n_seqs", [1, 8, 256])
@pytest.mark.parametrize("tokens", [1, 8, 20, 32, 50, 64, 100])
def test_a_workspace_for_the_table_is_enough_for_less(dtype, n_seqs, tokens):
    """What is asked for without a bound of the lengths does for every bound (which may choose
    another kernel)."""
    f = _lib.load().csdr_paged_attn_workspace_bytes
    for stride in (4, 64, 4096):
        c = kv(kv_dtype=dtype, n_seqs=n_seqs, table_stride=stride)
        n = n_seqs * tokens
        most = f(c, n, None, 0, 4, 0)
        for bound in (1, 16, 300, 1024, 1025, 5000, 40000, 65536):
            assert f(c, n, None, 0, 4, bound) <= most, (stride, bound)
