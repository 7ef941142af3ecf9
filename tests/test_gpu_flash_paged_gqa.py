"""GPU parity of flash_paged_gqa against softmax attention in 64 bits over the same pages.

Tolerance of an output element, from its roundings: the result to bf16 (2^-8 of it), every probability to bf16 (2^-8 of
sum_j p_j |v_j|), and the scores' error e (their products in fp32) and the exponential's, at most 2 (e + 2^-18) of the same
sum.  A weight under 2^-102 of its row's largest may be 0 (fp32 ends at 2^-126, and weights are held relative to 2^24 times
the largest): up to 2^16 such keys (the caches here have fewer) are 2^-86 of the largest value, 448 of the largest scale.
lse: e and a few units of fp32."""
import math

import pytest
import torch

from oracle import gqa
from tests import _gqa
from tilert_amd.flash_paged_gqa import flash_paged_gqa

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def run(cuda, q, pages, table, cu, lens, kv, **kw):
    out = torch.full(q.shape, 7.0, dtype=BF16, device=cuda)
    lse = torch.full(q.shape[:-1], 7.0, device=cuda)
    flash_paged_gqa(*_gqa.to(cuda, q, pages, table, cu, lens), out, lse, kv_heads=kv, **kw)
    torch.cuda.synchronize()
    return out, lse


def check(cuda, q, pages, table, cu, lens, kv, out, lse, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, want_lse, spread, slack = gqa.attention(*_gqa.to(cuda, q, pages, table, cu, lens), kv, scale)
    mine = torch.zeros_like(want_lse, dtype=torch.bool)
    mine[:int(cu[-1])] = True
    bad = mine[..., None] & torch.isnan(want)  # the definition gives NaN: a NaN in a key or value that is seen
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[mine & torch.isnan(want_lse)]).all()
    e = slack[..., None]
    tol = 2 ** -8 * want.abs() + (2 ** -8 + 2 * (e + 2 ** -18)) * spread
    scales = gqa.views(pages, kv, q.shape[-1])[2][..., 1].double()
    tol = tol + 2.0 ** -86 * 448 * float(scales[(scales > 0) & (scales < 2.0 ** 127)].max())
    off = (out.double() - want).abs()
    fine = mine[..., None] & ~bad
    assert torch.all(off[fine] <= tol[fine]), (off[fine] / tol[fine].clamp_min(1e-300)).max()
    assert torch.all(out[~mine] == 7.0) and torch.all(lse[~mine] == 7.0)  # rows of no sequence
    seen = mine & torch.isfinite(want_lse)
    assert torch.all((lse.double() - want_lse).abs()[seen] <= (slack + 2 ** -20 * (1 + want_lse.abs()))[seen])
    blind = mine & torch.isneginf(want_lse)
    assert torch.isneginf(lse[blind]).all() and torch.all(out[blind] == 0)


CASES = [  # new tokens, cache lengths, heads, kv heads, dim, padding
    ([1], [1], 8, 8, 128, 0), ([1], [2], 1, 1, 64, 0), ([1], [63], 32, 8, 128, 1), ([1], [64], 20, 4, 64, 0), ([1], [65], 28, 4, 128, 0),
    ([1], [500], 32, 8, 128, 0), ([1], [129], 128, 1, 128, 0), ([1], [700], 24, 1, 64, 3), ([4], [4], 64, 8, 128, 0), ([4], [300], 16, 2, 64, 2),
    ([7], [70], 3, 3, 128, 0), ([33], [40], 10, 2, 128, 0), ([1], [4000], 16, 2, 128, 0), ([2], [5000], 128, 2, 64, 0), ([257], [700], 32, 8, 128, 5),
    ([64], [64], 20, 4, 64, 0), ([1, 1, 1], [10, 200, 64], 16, 4, 128, 0), ([1, 5, 0, 40, 1], [90, 5, 33, 400, 1], 40, 8, 128, 3),
    ([0, 0, 3], [0, 9, 64], 8, 2, 64, 1), ([1] * 70, list(range(1, 211, 3)), 16, 2, 128, 4), ([100, 1, 1], [130, 3000, 1], 20, 5, 128, 0),
    ([1] * 5, [64 * i for i in range(1, 6)], 128, 8, 128, 0), ([500], [1500], 8, 1, 128, 0), ([1], [40000], 16, 2, 128, 0),
    ([3], [30000], 8, 1, 64, 0), ([700, 300], [2000, 2500], 16, 2, 128, 0), ([1] * 40, [100 * i + 1 for i in range(40)], 32, 4, 64, 0),
    ([300, 1, 129], [300, 900, 640], 8, 8, 64, 2), ([2, 17], [3000, 65], 96, 1, 128, 0),
]


@pytest.mark.parametrize("new,total,heads,kv,dim,pad", CASES)
def test_against_64_bits(cuda, new, total, heads, kv, dim, pad):
    print("case", new[:8], total[:8], heads, kv, dim, pad, flush=True)
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, pad=pad, extra_columns=1, seed=sum(total) + heads)
    _gqa.fill(pages, table, total, kv, dim)
    q = _gqa.queries(rows, heads, dim, 21)
    out, lse = run(cuda, q, pages, table, cu, lens, kv)
    check(cuda, q, pages, table, cu, lens, kv, out, lse)


@pytest.mark.parametrize("std", [0.02, 6.0])
def test_flat_and_peaked_softmax(cuda, std):
    pages, table, cu, lens, rows = _gqa.batch([3, 200], [600, 900], 2, 128, seed=23)
    _gqa.fill(pages, table, [600, 900], 2, 128, std=2.0, spread=2.0)
    q = _gqa.queries(rows, 8, 128, 25, std)
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    check(cuda, q, pages, table, cu, lens, 2, out, lse)


@pytest.mark.parametrize("new", [2, 150])
def test_scores_that_grow_along_the_cache(cuda, new):
    """Every page raises the running maximum: the sums so far are rescaled again and again."""
    total, kv, dim = [1500, 1400], 2, 64
    pages, table, cu, lens, rows = _gqa.batch([new, 40], total, kv, dim, seed=27)
    _gqa.fill(pages, table, total, kv, dim)
    k, _, scales = gqa.views(pages, kv, dim)
    for b, n in enumerate(total):  # keys that agree with every query, growing with the position
        p = torch.arange(n)
        page = table[b].long()[p // 64]
        scales[page, :, 0] = 2.0 ** -6
        k[page, :, p % 64] = _gqa.codes_of(p[:, None, None] / 400.0, 2.0 ** -6).expand(n, kv, dim)
    q = torch.full((rows, 8, dim), 0.5, dtype=BF16)
    out, lse = run(cuda, q, pages, table, cu, lens, kv, scale=0.7)
    check(cuda, q, pages, table, cu, lens, kv, out, lse, 0.7)


@pytest.mark.parametrize("new", [1, 200])
def test_a_heavy_key_in_front_of_a_flat_tail(cuda, new):
    """One key holds most of a row's weight and has values of 0; thousands of far lighter ones make the result together."""
    total, kv, dim = [6000], 1, 128
    pages, table, cu, lens, rows = _gqa.batch([new], total, kv, dim, seed=67)
    _gqa.fill(pages, table, total, kv, dim)
    k, v, scales = gqa.views(pages, kv, dim)
    page = int(table[0, 0])
    scales[page, 0, 0] = 1.0
    k[page, 0, 1:] = 0
    k[page, 0, 0] = _gqa.codes_of(torch.full((dim,), 1.0), 1.0)
    v[page, 0, :, 0] = 0
    q = torch.full((rows, 8, dim), 1.25, dtype=BF16)
    out, lse = run(cuda, q, pages, table, cu, lens, kv)
    check(cuda, q, pages, table, cu, lens, kv, out, lse)


@pytest.mark.parametrize("new,size", [(1, 2.0 ** 119), (100, 2.0 ** 119), (1, 2.0 ** -20), (100, 2.0 ** -20)])
def test_values_at_the_ends_of_the_scales(cuda, new, size):
    """Values near the largest of bf16, whose plain sum passes fp32, and near the least scale's."""
    total, kv, dim = [3000], 2, 64
    pages, table, cu, lens, rows = _gqa.batch([new], total, kv, dim, seed=69)
    _gqa.fill(pages, table, total, kv, dim)
    k, v, scales = gqa.views(pages, kv, dim)
    used = table[0].long()
    scales[used, :, 1] = size
    v[used] = v[used] & 0x77  # (positive, at most 240)
    q = _gqa.queries(rows, 8, dim, 71, 0.5)
    out, lse = run(cuda, q, pages, table, cu, lens, kv)
    check(cuda, q, pages, table, cu, lens, kv, out, lse)


@pytest.mark.parametrize("heads", [4, 64])
def test_tokens_that_see_nothing(cuda, heads):
    """More new tokens than keys: the first ones stand before position 0."""
    pages, table, cu, lens, rows = _gqa.batch([6, 3], [6, 3], 2, 128, seed=31)
    _gqa.fill(pages, table, [6, 3], 2, 128)
    lens[0], lens[1] = 2, -4
    q = _gqa.queries(rows, heads, 128, 33)
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    check(cuda, q, pages, table, cu, lens, 2, out, lse)
    assert torch.isneginf(lse[:4]).all() and torch.isfinite(lse[4:6]).all() and torch.isneginf(lse[6:]).all()


@pytest.mark.parametrize("new", [1, 150])
def test_pages_outside_the_pool_are_not_seen(cuda, new):
    pages, table, cu, lens, rows = _gqa.batch([new, new, new], [300, 200, 150], 2, 64, seed=35)
    _gqa.fill(pages, table, [300, 200, 150], 2, 64)
    table[0, 1], table[0, 4], table[1, 0], table[2, :3] = -1, pages.shape[0], 2 ** 31 - 1, -7
    table[2, 0] = -2 ** 31
    lens[1] = 400  # 200 positions past the table
    q = _gqa.queries(rows, 16, 64, 37)
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    check(cuda, q, pages, table, cu, lens, 2, out, lse)
    assert torch.isneginf(lse[2 * new:]).all()


@pytest.mark.parametrize("new", [1, 4, 200])
def test_bad_pages_among_many(cuda, new):
    """Enough pages that a workgroup takes several, bad ones first, last and between them, also the first pages of a cache."""
    total = [4000, 5000, 3500] if new > 4 else [12000, 9000, 15000]
    pages, table, cu, lens, rows = _gqa.batch([new] * 3, total, 2, 64, seed=59)
    _gqa.fill(pages, table, total, 2, 64)
    g = torch.Generator().manual_seed(61)
    for b, n in enumerate(total):
        need = -(-n // 64)
        bad = torch.randperm(need, generator=g)[:need // 3]
        table[b, bad] = torch.where(bad % 2 == 0, -2, pages.shape[0]).to(torch.int32)
        table[b, :4] = -2
    table[2, :-(-total[2] // 64) - 1] = -3  # one page is left, the last
    pages, table = torch.cat([torch.full_like(pages[:1], 0xff), pages]), table + 1  # page 0 is nobody's, and NaN
    q = _gqa.queries(rows, 8, 64, 63)
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    check(cuda, q, pages, table, cu, lens, 2, out, lse)


@pytest.mark.parametrize("new", [1, 150])
def test_a_cache_longer_than_its_table(cuda, new):
    """Positions past the table's columns hold no key: the tokens see the table's, all of them."""
    pages, table, cu, lens, rows = _gqa.batch([new, new], [320, 320], 2, 128, seed=55)
    _gqa.fill(pages, table, [320, 320], 2, 128)
    lens[0], lens[1] = 320 + 7, 2 ** 31 - 1
    q = _gqa.queries(rows, 8, 128, 57)
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    check(cuda, q, pages, table, cu, lens, 2, out, lse)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("what", ["key", "value", "key scale", "value scale", "infinite scale", "negative scale"])
@pytest.mark.parametrize("new,total,back", [(50, 250, 30), (300, 430, 30), (300, 430, 100), (300, 430, 50)])
def test_a_bad_key_reaches_only_the_tokens_that_see_it(cuda, what, new, total, back):
    """A NaN in a key's or value's codes, or a scale that is none: tokens before it are as without it, bit for bit, and
    those from it on are NaN where the definition is."""
    pages, table, cu, lens, rows = _gqa.batch([new], [total], 2, 128, seed=39)
    _gqa.fill(pages, table, [total], 2, 128)
    q = _gqa.queries(rows, 8, 128, 41)
    clean, clean_lse = run(cuda, q, pages, table, cu, lens, 2)
    at = total - back
    page, row, first = int(table[0, at // 64]), at % 64, at - (total - new)
    k, v, scales = gqa.views(pages, 2, 128)
    if what == "key":
        k[page, 1, row, 100] = 0x7f
    elif what == "value":
        v[page, 1, 100, row] = 0xff
    else:
        scales[page, 1, 0 if what == "key scale" else 1] = {"infinite scale": math.inf, "negative scale": -1.0}.get(what, math.nan)
        first = max(first - row, 0)
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    assert torch.equal(out[:first], clean[:first]) and torch.equal(lse[:first], clean_lse[:first])
    assert torch.equal(out[:, :4], clean[:, :4])  # the other kv head
    check(cuda, q, pages, table, cu, lens, 2, out, lse)
    assert torch.isnan(out[first:, 4:, 100]).all()


@pytest.mark.parametrize("new", [3, 200])
def test_a_bad_query_reaches_only_its_row(cuda, new):
    pages, table, cu, lens, rows = _gqa.batch([new], [500], 2, 64, seed=73)
    _gqa.fill(pages, table, [500], 2, 64)
    q = _gqa.queries(rows, 8, 64, 75)
    clean, clean_lse = run(cuda, q, pages, table, cu, lens, 2)
    q[1, 2, 5], q[1, 7, 6] = math.nan, math.inf
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    bad = torch.zeros(rows, 8, dtype=torch.bool, device=cuda)
    bad[1, 2] = bad[1, 7] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[1, 2])
    assert torch.equal(out[~bad], clean[~bad]) and torch.equal(lse[~bad], clean_lse[~bad])


def test_repeats_are_equal_bit_for_bit(cuda):
    pages, table, cu, lens, rows = _gqa.batch([1, 130, 1], [5000, 400, 77], 2, 128, seed=43)
    _gqa.fill(pages, table, [5000, 400, 77], 2, 128)
    q = _gqa.queries(rows, 16, 128, 45)
    first = run(cuda, q, pages, table, cu, lens, 2)
    for _ in range(3):
        again = run(cuda, q, pages, table, cu, lens, 2)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("new", [4, 150])
def test_a_strided_query_and_no_lse(cuda, new):
    pages, table, cu, lens, rows = _gqa.batch([new], [390], 2, 128, seed=47)
    _gqa.fill(pages, table, [390], 2, 128)
    joint = _gqa.queries(rows, 12, 128, 49).to(cuda)
    q = joint[:, 4:12]
    want, _ = run(cuda, q.contiguous(), pages, table, cu, lens, 2)
    out = torch.zeros(rows, 8, 128, dtype=BF16, device=cuda)
    flash_paged_gqa(q, *_gqa.to(cuda, pages, table, cu, lens), out, kv_heads=2)
    assert torch.equal(out, want)


def test_no_tokens(cuda):
    pages, table, cu, lens, _ = _gqa.batch([0], [5], 2, 64, seed=51)
    out, lse = run(cuda, _gqa.queries(0, 8, 64, 53), pages, table, cu, lens, 2)
    assert out.numel() == 0 and lse.numel() == 0
