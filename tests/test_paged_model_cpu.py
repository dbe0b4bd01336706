"""What of paged serving needs no GPU: a time limit that is refused."""
import pytest

from test_paged_cpu import attention_args, ops


@pytest.mark.parametrize("timeout_ms", [0, -1, 60001])
def test_attention_refuses_a_time_limit(timeout_ms):
    with pytest.raises(RuntimeError, match="timeout_ms"):
        ops().paged_attention(**attention_args(), timeout_ms=timeout_ms)
