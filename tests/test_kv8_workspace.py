"""The workspace of the 8-bit cache's attention stays small, whatever the rows, samples and blocks."""
import itertools

import pytest

from flashact_amd import _lib


@pytest.mark.parametrize("hd", [64, 96, 128, 256])
def test_workspace_is_bounded(hd):
    """At most 4096 sums of 16 rows, and 16 words of 8 bytes for each tile of rows that is split."""
    need = _lib.lib().fa_kv8_attention_workspace_bytes
    most = 0
    for batch, tokens, heads, blocks in itertools.product((1, 2, 5, 16, 65), (1, 33, 257, 1025, 2049, 8200), (1, 8, 24),
                                                          (1, 7, 64, 300, 4096, 1 << 20)):
        for kv_heads in (1, heads):
            most = max(most, need(batch, tokens, heads, kv_heads, hd, blocks))
    assert 0 < most <= 4096 * ((16 * hd + 32) * 4 + 16 * 8) + 256
    assert need(1, 1, 8, 1, hd, 4096) > 0  # few rows over many keys are split
