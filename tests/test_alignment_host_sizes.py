"""Sizes at the ends of what the alignment operators take, without a GPU: workspace queries and refusals in front of any launch."""
import pytest

from fastspeech2_amd import hip

GB = 1 << 30


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
