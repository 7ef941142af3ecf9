"""The paged attention's plan and the paged operators' limits at the sizes where 32-bit arithmetic ends: on the CPU, through
the C entries, which refuse or plan before any launch."""
import pytest

from tests.test_paged_checks import ENTRIES, _attend_c, _read_c, _refused, _write_c
from tilert_amd import _lib

TILES = 2048  # row tiles that a split launch plans at most
START = 10    # units that a tile counts for besides its pages
WGS = 256     # workgroups, each with ceil(units / WGS) units


@pytest.mark.parametrize("tokens,heads,rows", [(8188, 16, 64), (8180, 16, 64), (2 ** 14, 8, 64), (1023, 128, 64), (1, 16, 16)])
def test_a_split_launch_counts_its_units_in_31_bits(tokens, heads, rows):
    """One sequence whose tiles all see a table of `pages`: where their units, and the end of the last workgroup's share of
    them, would pass 2^31 - 1, the tiles are not split (no workspace)."""
    f = _lib.load().tl_flash_paged_mla_workspace_bytes
    tiles = tokens * heads // rows + 1
    for pages in (9, 2 ** 16, 2 ** 20 - 12, 2 ** 20 - 11, 2 ** 20 - 10, 2 ** 20):
        units = tiles * (pages + START)
        quota = -(-units // WGS)
        fits = tiles <= TILES and max(units, WGS * quota) < 2 ** 31
        assert (f(1, tokens, heads, pages) > 0) == fits, (tiles, pages)


# A launch has fewer than 2^32 threads: a wave a token, in workgroups of four tokens.  The null pointers are asked for behind the
# sizes, so that nothing is launched on either side of the border.
@pytest.mark.parametrize("tokens", [2 ** 26 - 3, 2 ** 26 - 1])
@pytest.mark.parametrize("name,args", ENTRIES)
def test_more_tokens_than_a_launch_has_waves(name, args, tokens):
    assert -(-tokens // 4) * 256 >= 2 ** 32
    null = dict(q=None, heads=1) if args is _attend_c else dict(kv=None)
    _refused(name, args(n_tokens=tokens, **null), 1, "out of range")


@pytest.mark.parametrize("name,args", [("tl_mla_cache_write", _write_c), ("tl_mla_cache_read", _read_c)])
def test_the_most_tokens_of_a_launch(name, args):
    tokens = 2 ** 26 - 4
    assert -(-tokens // 4) * 256 < 2 ** 32
    _refused(name, args(n_tokens=tokens, kv=None), 1, "null pointer")
