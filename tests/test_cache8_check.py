"""The attention over the 8-bit cache without a GPU: what b200k_cache8_attention_check refuses before any call of the device,
and scratch sizes that serve smaller calls."""
import ctypes

import pytest

from b200fwd import abi
from test_cache8 import lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("scratch", [None, (1 << 20) + 16])
def test_cache8_attention_check_refusals(lib, scratch):  # noqa: F811
    assert lib.b200k_cache8_attention_check(scratch, None) == abi.EINVAL
    assert "256-byte" in abi.last_error()


@pytest.mark.parametrize("heads,nkv", [(32, 8), (8, 8), (71, 1), (16, 2)])
@pytest.mark.parametrize("half", [0, 1])
def test_cache8_attention_scratch_serves_smaller_calls(lib, heads, nkv, half):  # noqa: F811
    """Never less for more tokens or more requests (a program sizes it once, for the most of both)."""
    size = ctypes.c_uint64()

    def of(n, n_seqs):
        assert lib.b200k_cache8_attention_scratch(n, n_seqs, heads, nkv, 64, half, ctypes.byref(size)) == 0
        return size.value

    steps = [1, 2, 3, 5, 8, 15, 16, 17, 31, 33, 64, 65, 100, 128, 129, 256, 257, 1000, 4096]
    for n in steps:
        by_seqs = [of(n, s) for s in steps]
        assert by_seqs == sorted(by_seqs)
    for s in steps:
        by_n = [of(n, s) for n in steps]
        assert by_n == sorted(by_n)
