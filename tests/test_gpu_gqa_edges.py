"""The paged per-head cache's operators where rows, blocks and sizes meet their ends."""
import pytest
import torch

from oracle import gqa
from tests import _gqa
from tests.test_gpu_flash_paged_gqa import check, run

pytestmark = pytest.mark.gpu
U8 = torch.uint8


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,total", [(3, 700), (100, 1500), (100, 500)])  # few rows; many, their pages cut and whole
@pytest.mark.parametrize("what", ["query", "key"])
def test_a_row_follows_from_what_it_sees_alone(cuda, what, new, total, dim):
    """One row whose maximum leaps from page to page, among rows whose maximum rises a little: the others are as without it, bit
    for bit."""
    pages, table, cu, lens, rows = _gqa.batch([new], [total], 2, dim, seed=131)
    _gqa.fill(pages, table, [total], 2, dim)
    q = _gqa.queries(rows, 8, dim, 133)
    clean, clean_lse = run(cuda, q, pages, table, cu, lens, 2)
    other = torch.ones(rows, 8, dtype=torch.bool, device=cuda)
    if what == "query":
        for t, h in ((1, 2), (rows - 1, 5)):
            q[t, h] *= 16
            other[t, h] = False
    else:  # the last token's own key, in line with one of its queries: 448 of its block's scale in each dim
        k, _, _ = gqa.views(pages, 2, dim)
        k[int(table[0, (total - 1) // 64]), 1, (total - 1) % 64] = torch.where(q[-1, 6] < 0, 0xfe, 0x7e).to(U8)
        other[-1, 4:] = False
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    assert torch.equal(out[other], clean[other]) and torch.equal(lse[other], clean_lse[other])
    check(cuda, q, pages, table, cu, lens, 2, out, lse)
