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


@pytest.mark.parametrize("dt", [_lib.FM_BF16, _lib.FM_F32])
@pytest.mark.parametrize("d", [64, 96, 128, 256])
def test_pieces_need_no_large_workspace(dt, d):
    lib = _lib.load()
    for H, G in ((1, 1), (1, 8), (8, 8), (64, 1)):
        for S, L in ((1, 1), (1, 1 << 20), (512, 512), (4096, 4096), (1 << 20, 32)):
            rows, keys = H * G * S, H * L
            # pieces: fp32 rows of at most 512 + H G blocks of 128 queries; splits: two of at most 1024 + H blocks of 128 keys
            small = 40 * (rows + keys) + (1 << 20)             # masks, {lse, D}, norms
            assert 0 < lib.fm_local_attn_terms_fwd_workspace(H, G, S, L, d, dt) <= small + 2 * (512 + H * G) * 128 * (d + 2) * 4
            assert 0 < lib.fm_local_attn_terms_bwd_workspace(H, G, S, L, d, dt) <= \
                small + 2 * (512 + H * G) * 128 * d * 4 + 2 * (1024 + H) * 2 * 128 * d * 4


def test_a_page_of_no_tokens_is_refused():
    from fast_memory_amd import PagedCache
    for page in (0, -4):
        with pytest.raises(ValueError):
            PagedCache(1, 4, page, 1, 64, device="cpu", max_tokens=8)
