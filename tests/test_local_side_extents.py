"""Workspaces of the local side by extents alone (no GPU)."""
import pytest

from fast_memory_amd import _lib


@pytest.mark.parametrize("dt", [_lib.FM_BF16, _lib.FM_F16, _lib.FM_F32])
@pytest.mark.parametrize("d", [64, 128, 256, 96])
def test_a_cache_of_many_rows_needs_no_large_workspace(dt, d):
    """A call of few tokens over a cache of many rows: what it needs follows the tokens, not the rows."""
    lib = _lib.load()
    for rows in (1, 64, 2048, 65536):
        for T, max_new in ((1, 1), (1, 0), (4, 0), (70, 0), (70, 64), (rows, 1)):
            for H, G in ((8, 8), (1, 1), (1, 64), (64, 1)):
                if T * H * G > 1 << 22:
                    continue
                need = lib.fm_paged_attn_fwd_workspace(rows, T, max_new, H, G, d, 2048, 16, dt)
                # pieces until there are about 1024 workgroups of at most 128 query rows, twice over where ceilings add up, or
                # one piece; d + 2 words a unit
                assert 0 < need <= 2 * 2 * (1024 + H) * 128 * (d + 2) * 4, (rows, T, max_new, H, G)
