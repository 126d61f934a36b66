"""Sizes at the ends of what the alignment operators take, without a GPU: workspace queries and refusals in front of any launch."""
import pytest

from fastspeech2_amd import hip
from tests.test_alignment_host import _norm

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
