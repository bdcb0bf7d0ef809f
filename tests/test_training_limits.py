"""Sizes beyond what the attention's gradient can count are refused before anything is launched (CPU only)."""

import pytest

from kernel_opt_agent_b200 import _lib
from tests.test_training_capi import OK, P, UNSUPPORTED


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sq,skv", [(2 ** 31 - 1, 128), (128, 2 ** 31 - 1), (2 ** 31 - 127, 2 ** 31 - 127)])
def test_sequences_whose_tiles_pass_31_bits(d, sq, skv):
    """Rounded up to whole tiles such a length leaves int's range (a workspace that large is only claimed here)."""
    rc = _lib.load().tokmix_fa2_bwd(P, P, P, P, P, P, P, P, P, 1, 1, 1, sq, skv, d, 0, 0, 0.1, P, 1 << 62, None, None)
    assert rc == UNSUPPORTED and "tokens" in _lib.last_error()
    # no sequences: nothing to count
    assert _lib.load().tokmix_fa2_bwd(P, P, P, P, P, P, P, P, P, 0, 1, 1, sq, skv, d, 0, 0, 0.1, P, 1 << 62, None, None) == OK
