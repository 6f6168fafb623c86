"""Which calls of a text stage's operators take scratch for what (no GPU)."""

import ctypes as C

import pytest

from vllm_omni_amd import _lib


@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("causal", [0, 1])
def test_the_keys_lengths_are_taken_where_they_can_leave_tiles_out(cap, causal):
    """With slopes, from 6144 keys on; not where a window of less than a quarter of them leaves out more than the bound would."""
    def lengths_taken(S, window):
        need = [_lib.load().odit_attn_ruled_workspace_bytes(1, S, S, 32, 128, C.byref(_lib.AttnRules(causal=causal, window=window, cap=cap, slopes=slopes)))
                for slopes in (None, 1 << 20)]  # (the address is not read)
        assert need[1] - need[0] in (0, 32 * 64 * 4)
        return need[1] > need[0]

    assert lengths_taken(8192, 0) and lengths_taken(6144, 0) and not lengths_taken(6143, 0)
    assert lengths_taken(8192, 2048) and lengths_taken(8192, 1 << 30) and not lengths_taken(8192, 2047)
    assert not lengths_taken(8192, 1) and not lengths_taken(1 << 17, 4096)
