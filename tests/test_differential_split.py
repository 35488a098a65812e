"""The even split of a differential prefill, with the prices of its kernels:
every tile taken once, and every cut item's pieces found by the merge
(tests/host/prefill_split_check.h, on the CPU)."""
import pytest

from tests.test_stream_split import _run_host_check


@pytest.mark.parametrize("kernel", ["diff_prefill_split_check", "diff_prefill_split_f32_check"])
def test_prefill_split_invariants(kernel):
    _run_host_check(kernel)
