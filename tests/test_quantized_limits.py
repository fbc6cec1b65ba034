"""Sizes that the 8-bit calls refuse on the host because their kernels would count past 31 bits."""
import pytest

from shardserve_b200 import _native
from test_quantized_host import attend


@pytest.mark.parametrize("cols,kv_heads", [(1 << 26, 32), ((1 << 31) // 17 + 1, 17), ((1 << 27) - 1, 64)])
def test_attention_refuses_tables_past_31_bits(cols, kv_heads):
    assert attend(cols=cols, KVH=kv_heads, H=kv_heads) == _native.SS_ERR_INVALID
    assert "columns times kv_heads" in _native.last_error()


@pytest.mark.parametrize("cols,kv_heads", [((1 << 26) - 1, 32), ((1 << 31) // 17, 17), ((1 << 27) - 1, 16)])
def test_attention_takes_tables_up_to_31_bits(cols, kv_heads):
    """The next check, of the workspace, is reached."""
    assert attend(cols=cols, KVH=kv_heads, H=kv_heads, ws=None) == _native.SS_ERR_WORKSPACE
