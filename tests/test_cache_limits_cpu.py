"""The paged 8-bit cache's C ABI without a GPU: what its documents promise of sizes."""

from __future__ import annotations

import pytest

from fused_attn import abi

needs_lib = pytest.mark.skipif(not abi.available(), reason="libfa_sm100.so not built")

P16 = 0x1000


@needs_lib
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H", [1, 2, 4, 16])
@pytest.mark.parametrize("n_seqs", [1, 3, 64])
def test_a_workspace_serves_every_smaller_call(D, H, n_seqs):
    c = abi.FaCache(P16, P16, P16, P16, 8, 16, 1, D, (16 * D, 16 * D, D), (16 * D, 16 * D, D), P16, 4, 4, P16, P16,
                    n_seqs)
    sizes = [abi.cache_attention_workspace_bytes(c, H, T) for T in range(1, 70 * n_seqs)]
    assert all(0 < a <= b for a, b in zip(sizes, sizes[1:]))
    assert sizes[-1] > sizes[0]
