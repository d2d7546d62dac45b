"""Refusals of the windowed attention beyond those of test_fp8_window_args, without a GPU."""
import pytest

from test_fp8_window_args import ATT, I3, P


@pytest.mark.parametrize("name", ["ql", "kl"])
@pytest.mark.parametrize("by", [1, 2, 3])
def test_lengths_off_their_alignment_are_refused(lib, name, by):
    """The kernels read lengths as 4-byte integers; any other address would fault there."""
    a = {**ATT, "ql": P, "kl": P, name: P + by}
    assert lib.da3b_attention_window(*[I3(*v) if isinstance(v, tuple) else v for v in a.values()], None) == -1
