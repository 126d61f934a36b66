"""Sizes at the ends of what the alignment operators take, without a GPU: workspace queries and refusals in front of any launch."""
import pytest

from fastspeech2_amd import hip
from tests.test_alignment_host import _back, _mass, _norm

LONG = (1 << 31) - 1


@pytest.mark.parametrize("dtype", [0, 1])
def test_workspace_goes_by_the_rows_at_work(dtype):
    """one short utterance inside a large matrix asks for no more than in one of its own"""
    lib = hip.load()
    big = 100_000_000
    for B, q, k in ((1, 1, 65000), (1, 120, 4000), (3, 1, 2000)):
        n = lib.fs2_cross_attention_workspace(B, q, k, B * q, 2, 2, 128, dtype)
        assert 0 < n == lib.fs2_cross_attention_workspace(B, q, k, big, 2, 2, 128, dtype)
        assert n <= 256 * B * q * 2 * 130 * 4
    n = lib.fs2_cross_attention_bwd_workspace(1, 3000, 40, 3000, 40, 2, 2, 128, dtype)
    assert n > 4 * 2 * 3000 and n == lib.fs2_cross_attention_bwd_workspace(1, 3000, 40, 3000, big, 2, 2, 128, dtype)
    n = lib.fs2_cross_attention_mass_workspace(1, 3000, 40, 40, 2, 2, 128, dtype)
    assert 0 < n == lib.fs2_cross_attention_mass_workspace(1, 3000, 40, big, 2, 2, 128, dtype)


@pytest.mark.parametrize("change", [
    dict(B=1, H=1, KV=1, dk=32, ldq=32, ldk=32, ldv=32, ldo=32, max_k=1 << 30, Mk=1 << 30, dtype=1),
    dict(B=1, H=1, KV=1, dk=32, ldq=32, ldk=32, ldv=32, ldo=32, max_k=1 << 28, Mk=1 << 28, dtype=0),
    dict(B=8, H=1, KV=1, dk=32, ldq=32, ldk=32, ldv=32, ldo=32, max_k=1 << 26, Mk=1 << 30, dtype=1)])
def test_mass_refuses_more_work_items_than_a_launch_has(change):
    """512 work items for every 64 (fp32: 32) keys: 2^32 of them, or more, are no launch"""
    with pytest.raises(hip.HipError, match="in one launch"):
        _mass(change)


def test_backward_refuses_more_work_items_than_a_launch_has():
    """delta takes 16 rows and two heads to 256 work items: 2^28 rows of one head would be 2^32 of them"""
    with pytest.raises(hip.HipError, match="in one launch"):
        _back(dict(B=256, H=1, KV=1, max_q=1 << 20, Mq=1 << 20))


def test_group_norm_of_the_longest_utterance():
    """max_len up to 2^31 - 1 is planned in chunks (not taken for a short one where 32 bits overflow)"""
    lib = hip.load()
    for B, C, G in ((1, 8, 1), (1, 256, 16)):
        n = lib.fs2_group_norm_workspace(B, LONG, C, G)
        assert n > lib.fs2_group_norm_workspace(B, LONG // 2, C, G) > 0
        assert lib.fs2_group_norm_bwd_workspace(B, LONG, C, G) > lib.fs2_group_norm_bwd_workspace(B, LONG // 2, C, G)
    with pytest.raises(hip.HipError, match="fs2_group_norm_workspace"):
        hip.call("fs2_group_norm", *_norm(B=1, max_len=LONG, M=LONG, C=8, G=1, ldx=8, ldo=8, ws=None).values(), 0)
    with pytest.raises(hip.HipError, match="too many workgroups"):
        hip.call("fs2_group_norm", *_norm(B=1, max_len=LONG, M=LONG, C=1024, G=1, ldx=1024, ldo=1024).values(), 0)
