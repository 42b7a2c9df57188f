"""Limits of libmi_cache.so's attention that its sizes run into (CPU: nothing is launched)."""
import pytest

from test_cache_boundary import _attend, last


@pytest.mark.parametrize("max_kv", [(1 << 31) - 1, (1 << 31) - 8192])
def test_lengths_whose_steps_would_pass_32_bits(max_kv):
    assert _attend(max_kv=max_kv) == 2
    assert "max_kv_len" in last()


def test_lengths_up_to_there():
    assert _attend(max_kv=(1 << 31) - 8193) == 3      # (no workspace given)
