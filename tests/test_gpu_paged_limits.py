"""flash_paged_mla at the ends of its ranges: the widest tables, the smallest scales, the largest keys.  The tolerance is that of
test_gpu_paged_weights."""
import pytest
import torch

from oracle import paged
from tests import _paged
from tests.test_gpu_flash_paged_mla import queries, run
from tests.test_gpu_paged_weights import TILES, check_all, close, put
from tilert_amd.flash_paged_mla import flash_paged_mla

pytestmark = pytest.mark.gpu
ARCH = "deepseek_v3_2"
BF16, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("columns", [2 ** 20 - 11, 2 ** 20])
def test_the_most_tiles_over_the_widest_table(cuda, columns):
    """2048 row tiles: split with the one table, one workgroup a tile with the other."""
    g = torch.Generator(device=cuda).manual_seed(3)
    tokens, keys = 8188, 8300
    n = -(-keys // 64)
    pages = torch.empty(n, paged.PAGE_BYTES, dtype=torch.uint8, device=cuda)
    ids = torch.full((columns,), -1, dtype=I32, device=cuda)
    ids[:n] = torch.randperm(n, generator=g, device=cuda).to(I32)
    put(pages, ids, torch.randn(keys, 512, generator=g, device=cuda), torch.randn(keys, 64, generator=g, device=cuda))
    q, qp = ((torch.randn(tokens, 16, w, generator=g, device=cuda) * 0.3).to(BF16) for w in (512, 64))
    out, lse = torch.full_like(q, 7.0), torch.full((tokens, 16), 7.0, device=cuda)
    cu, lens = torch.tensor([0, tokens], dtype=I32, device=cuda), torch.tensor([keys], dtype=I32, device=cuda)
    flash_paged_mla(q, qp, pages, ids[None], cu, lens, out, lse, model_arch=ARCH)
    close(out, lse, q, qp, pages, ids, keys - tokens, [0, 1, 4000, tokens - 1])
    assert not (lse == 7.0).any()


def _case(cuda, new, total, heads, seed):
    pages, table, cu, lens, rows = _paged.batch([new], [total], seed=seed)
    _paged.fill(pages, table, [total], seed=seed)
    return list(_paged.to(cuda, *queries(rows, heads, seed + 1), pages, table, cu, lens))


@pytest.mark.parametrize("scale", [1e-6, 1e-12, 1e-30, 2.0 ** -126])
@pytest.mark.parametrize("new,heads", TILES)
@pytest.mark.parametrize("total", [90, 1000])
def test_zero_queries_and_a_tiny_scale(cuda, new, heads, total, scale):
    """All keys weigh alike, on whole and on masked pages: a score's factor, the row's power of two times the scale, may be
    below fp32's numbers, and a masked score is still -inf."""
    case = _case(cuda, new, total, heads, 5)
    case[0][:, ::2] = 0
    case[1][:, ::2] = 0
    case[0][:, 1::4] *= 2.0 ** -100
    case[1][:, 1::4] *= 2.0 ** -100
    out, lse = run(cuda, *case, scale=scale)
    check_all(case, out, lse, scale)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("size", [1e30, 1e38])
@pytest.mark.parametrize("new,heads", TILES)
@pytest.mark.parametrize("total", [300, 3000])  # one kernel; split and joined
def test_keys_near_the_largest_numbers(cuda, new, heads, total, size):
    """Latents of one sign whose sums pass fp32's range while their means do not; no part of the scores is theirs."""
    g = torch.Generator().manual_seed(7)
    case = _case(cuda, new, total, heads, 9)
    case[0].zero_()
    latent = (1 + 0.2 * torch.randn(total, 512, generator=g).clamp(-3, 3)) * size
    put(case[2], case[3][0], latent.to(cuda), torch.randn(total, 64, generator=g).to(cuda))
    out, lse = run(cuda, *case)
    assert torch.isfinite(out).all()
    check_all(case, out, lse)


@pytest.mark.parametrize("power", [5, 8])
@pytest.mark.parametrize("new,heads", TILES)
@pytest.mark.parametrize("total", [200, 1500])
def test_one_dim_far_above_the_others(cuda, new, heads, total, power):
    """A dim whose latents are 2^power times the others', of one sign: its products are most of every score, and alike."""
    g = torch.Generator().manual_seed(11)
    case = _case(cuda, new, total, heads, 13)
    latent = torch.randn(total, 512, generator=g)
    latent[:, 77] = 2.0 ** power * (1 + 0.01 * torch.randn(total, generator=g))
    put(case[2], case[3][0], latent.to(cuda), torch.randn(total, 64, generator=g).to(cuda))
    out, lse = run(cuda, *case)
    check_all(case, out, lse, cut=True)
