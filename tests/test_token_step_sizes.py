"""Workspace sizes of prompt attention with modified scores: for any arguments."""
import pytest


@pytest.fixture(scope="module")
def ws(vsl):
    return vsl.hip().vsl_attn_prefill_mods_ws_bytes


@pytest.mark.parametrize("S,pos0,n_q,n_kv", [(0xFFFFFFFF, 0, 8, 2), (0xFFFFFFE1, 7, 1, 1), (0x80000000, 0, 256, 256),
                                             (0x80000000, 0xFFFFFFFF, 1 << 31, 1 << 31), (0xFFFFFFFF, 0xFFFFFFFF, 0xFFFFFFFF, 1),
                                             (0xFFFFFFE0, 0, 0xFFFFFFFF, 0xFFFFFFFF)])
def test_sizes_that_no_call_takes(ws, S, pos0, n_q, n_kv):
    """A number of blocks that does not fit 32 bits is many blocks, not none."""
    assert ws(S, pos0, n_q, n_kv, 128) == 0
