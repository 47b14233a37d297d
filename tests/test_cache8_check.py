"""b200k_cache8_attention_check without a GPU: what it refuses before any call of the device."""
import pytest

from b200fwd import abi
from test_cache8 import lib  # noqa: F401 (a fixture)


@pytest.mark.parametrize("scratch", [None, (1 << 20) + 16])
def test_cache8_attention_check_refusals(lib, scratch):  # noqa: F811
    assert lib.b200k_cache8_attention_check(scratch, None) == abi.EINVAL
    assert "256-byte" in abi.last_error()
