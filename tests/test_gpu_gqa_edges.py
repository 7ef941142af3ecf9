"""The paged per-head cache's operators where rows, blocks and sizes meet their ends."""
import math

import pytest
import torch

from oracle import gqa
from tests import _gqa
from tests.test_gpu_flash_paged_gqa import check, run
from tests.test_gpu_gqa_cache import check_sums, check_write, evict, evict_case, inputs, write
from tilert_amd.gqa_cache import gqa_cache_weights, gqa_cache_write

pytestmark = pytest.mark.gpu
BF16, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


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


def append(cuda, pages, table, lens, key, value, n):
    """The pages after a write of key and value behind the first n keys."""
    p = pages.to(cuda)
    cu = torch.tensor([0, key.shape[0]], dtype=I32)
    gqa_cache_write(*_gqa.to(cuda, key, value), p, *_gqa.to(cuda, table, cu, lens))
    return p.cpu()


@pytest.mark.parametrize("side", ["key", "value", "both"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -1.0, 0.0, 2.0 ** -127])
@pytest.mark.parametrize("old,new,dim,size", [(37, 3, 128, 1.0), (5, 1, 64, 100.0), (62, 2, 64, 0.01), (130, 70, 128, 1.0)])
def test_older_keys_under_no_scale_stay_nan(cuda, side, bad, old, new, dim, size):
    """New keys in a page whose older ones are NaN for a scale that is none: those stay NaN, keys and values, and the new ones are the
    block's only ones for its new scales; the other head's block and other pages are as they were."""
    pages, table, _, _, _ = _gqa.batch([new], [old + new], 2, dim, seed=141)
    _gqa.fill(pages, table, [old], 2, dim)
    lens = torch.tensor([old + new], dtype=I32)
    g = torch.Generator().manual_seed(143)
    key, value = ((torch.randn(new, 2, dim, generator=g) * size).to(BF16) for _ in range(2))
    clean = append(cuda, pages, table, lens, key, value, old)
    page, r0 = int(table[0, old // 64]), old % 64
    r1 = min(64, r0 + new)
    _, _, scales = gqa.views(pages, 2, dim)
    for i, name in enumerate(("key", "value")):
        if side in (name, "both"):
            scales[page, 1, i] = bad
    after = append(cuda, pages, table, lens, key, value, old)
    for got, want, x in zip(gqa.views(after, 2, dim), gqa.views(clean, 2, dim), (key, value, None)):
        same = torch.ones(pages.shape[0], 2, dtype=torch.bool)
        same[page, 1] = False
        assert torch.equal(got[same].view(U8), want[same].view(U8))
        if x is None:
            continue
        codes, i = (got[page, 1], 0) if x is key else (got[page, 1].T, 1)
        s = gqa.views(after, 2, dim)[2][page, 1, i]
        assert torch.isnan(gqa.value_of(codes[:r0])).all()
        assert float(s) == gqa.scale_of(float(x[:r1 - r0, 1].float().abs().max()))
        assert torch.equal(codes[r0:r1], _gqa.codes_of(x[:r1 - r0, 1].float(), s))
    q, cu = _gqa.queries(new, 4, dim, 145), torch.tensor([0, new], dtype=I32)
    out, lse = run(cuda, q, after, table, cu, lens, 2)
    check(cuda, q, after, table, cu, lens, 2, out, lse)
    assert torch.isnan(out[:, 2:]).all() and torch.isnan(lse[:, 2:]).all() and torch.isfinite(out[:, :2]).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("std", [1e18, 1e19, 1e30, 3e38])
@pytest.mark.parametrize("turn", [False, True])
def test_norms_of_rows_whose_squares_pass_fp32(cuda, turn, std, dim):
    new, total, kv = [70, 3], [100, 64], 2
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, seed=151)
    _gqa.fill(pages, table, [t - n for n, t in zip(new, total)], kv, dim)
    joint, gq, gk, freqs = inputs(rows, 4, kv, dim, 64, 153, 0.0)
    g = torch.Generator().manual_seed(155)
    joint = ((torch.rand(joint.shape, generator=g) * 2 - 1) * std).to(BF16)
    joint[1::3] = (joint[1::3].float() / std).to(BF16)  # every third token of ordinary rows
    joint[:, 4 + kv:] = torch.randn(rows, kv, dim, generator=g).to(BF16)
    freqs = freqs if turn else None
    after, out = write(cuda, joint, 4, kv, pages, table, cu, lens, gq, gk, freqs)
    check_write(pages, after, joint, 4, kv, dim, table, cu, lens, gq, gk, freqs, False, out)


@pytest.mark.parametrize("std,eps", [(1e-16, 0.0), (1e-30, 0.0), (1e-38, 0.0), (1e-38, 1e-38), (1e-30, 1e-45), (1e-20, 1e-12), (3e38, 0.0), (3e38, 1e30)])
def test_norms_with_a_small_or_large_eps(cuda, std, eps):
    """Rows of sizes whose squares fall below fp32 or pass it, with an eps that is as small, nothing, or far larger: within the
    roundings of a norm, 2^-20 (the writer's tests say of what), and of bf16."""
    dim, rows = 128, 40
    g = torch.Generator().manual_seed(157)
    q = ((torch.rand(rows, 4, dim, generator=g) * 2 - 1) * std).to(BF16)
    pages, table, cu, lens, _ = _gqa.batch([rows], [rows], 4, dim, seed=159)
    gamma, out = torch.rand(dim, generator=g) + 0.5, torch.zeros(rows, 4, dim, dtype=BF16, device=cuda)
    gqa_cache_write(*_gqa.to(cuda, q, q, pages, table, cu, lens), gamma.to(cuda), query=q.to(cuda), gamma_q=gamma.to(cuda), query_out=out, eps=eps)
    want = gqa.turned(q, gamma, None, False, float(torch.tensor(eps, dtype=F32)))
    assert torch.all((out.cpu().double() - want).abs() <= (2 ** -8 + 2 ** -19) * want.abs() + 2.0 ** -134)  # (bf16's least step, 2^-133)


def test_a_row_of_zeros_and_rows_that_are_not_finite(cuda):
    """0 / sqrt(eps) is 0; a NaN or an infinity makes a query's row what the formula gives, and a key NaN."""
    dim = 64
    q = torch.randn(8, 1, dim, generator=torch.Generator().manual_seed(161)).to(BF16)
    q[0], q[1, 0, 3], q[2, 0, 5], q[3, 0, 7] = 0, math.nan, math.inf, -math.inf
    q[3, 0, 9:] = 3e38
    pages, table, cu, lens, _ = _gqa.batch([8], [8], 1, dim, seed=163)
    gamma, out, p = torch.ones(dim), torch.zeros(8, 1, dim, dtype=BF16, device=cuda), pages.to(cuda)
    gqa_cache_write(*_gqa.to(cuda, q, q.nan_to_num(1.0, 1.0, 1.0)), p, *_gqa.to(cuda, table, cu, lens, gamma), query=q.to(cuda), gamma_q=gamma.to(cuda), query_out=out)
    want = gqa.turned(q, gamma, None, False, 1e-6)
    assert torch.equal(torch.isnan(out.cpu()), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert torch.all((out.cpu().double() - want).abs()[fine] <= ((2 ** -8 + 2 ** -19) * want.abs())[fine])
    keys = gqa.value_of(gqa.views(p.cpu(), 1, dim)[0][int(table[0, 0]), 0, :8])
    assert torch.all(keys[0] == 0) and torch.isnan(keys[1:4]).all() and torch.isfinite(keys[4:]).all()


@pytest.mark.parametrize("new,total", [(1, 1), (3, 70), (16, 700), (100, 100), (100, 700)])
@pytest.mark.parametrize("dim", [64, 128])
def test_codes_of_a_page_s_earlier_use(cuda, dim, new, total):
    """A reused page's codes of 448 behind the last key, under the scale of the largest values, which takes them past bf16: no row
    sees them, and none is changed by them."""
    pages, table, cu, lens, rows = _gqa.batch([new], [total], 2, dim, seed=171)
    pages.fill_(0x7e)
    _gqa.fill(pages, table, [total - new], 2, dim)
    g = torch.Generator().manual_seed(173)
    key, value = torch.randn(new, 2, dim, generator=g).to(BF16), torch.randn(new, 2, dim, generator=g).to(BF16)
    value[:, 1] = torch.where(value[:, 1] < 0, -1, 1) * 3.3e38
    after = append(cuda, pages, table, lens, key, value, total - new)
    assert float(gqa.views(after, 2, dim)[2][int(table[0, (total - 1) // 64]), 1, 1]) == 2.0 ** 120
    q = _gqa.queries(rows, 8, dim, 175)
    out, lse = run(cuda, q, after, table, cu, lens, 2)
    check(cuda, q, after, table, cu, lens, 2, out, lse)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("new", [3, 100])
@pytest.mark.parametrize("power,most,code", [(120, 0x77, 0x78), (121, 0x6f, 0x70), (124, 0x57, 0x58), (127, 0x3f, 0x40), (127, 0x3f, 0x7e)])
def test_a_value_past_bf16_reaches_only_the_tokens_that_see_it(cuda, power, most, code, new):
    """A code that a scale takes past bf16 (the least: `most` is the last that stays inside), in the page of the newest tokens: rows before it are as without it, bit for bit, rows from
    it on are not finite in its dim."""
    total, dim = 200, 64
    pages, table, cu, lens, rows = _gqa.batch([new], [total], 2, dim, seed=177)
    _gqa.fill(pages, table, [total], 2, dim)
    q = _gqa.queries(rows, 8, dim, 179)
    _, v, scales = gqa.views(pages, 2, dim)
    page, row = int(table[0, (total - 2) // 64]), (total - 2) % 64
    scales[page, 1, 1] = 2.0 ** power
    v[page, 1] &= 0x83  # (subnormal codes)
    v[page, 1, 5, row] = most
    clean, clean_lse = run(cuda, q, pages, table, cu, lens, 2)
    assert torch.isfinite(clean).all()
    v[page, 1, 5, row] = code
    out, lse = run(cuda, q, pages, table, cu, lens, 2)
    assert torch.equal(lse, clean_lse) and torch.equal(out[:-2], clean[:-2]) and torch.equal(out[:, :4], clean[:, :4])
    assert not torch.isfinite(out[-2:, 4:, 5]).any()
    out[-2:, 4:, 5] = clean[-2:, 4:, 5]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_under_no_scale_are_nan_after_an_eviction(cuda, dim, side):
    """One of a block's two scales is none: its keys are NaN in the attention and in the key weights, before an eviction and after it."""
    args = evict_case([300], [130], 2, dim, 181)
    pages, w, table, lens, keep, to = args
    bad = int(table[0, 1])
    gqa.views(pages, 2, dim)[2][bad, 1, side] = math.nan
    w[bad, 1, 5:20] = 1e9  # some of them stay
    after, _, kept, slots = evict(cuda, *args, 2, dim, 30)
    mine = slots[0, 1]
    from_bad = (mine >= 64) & (mine < 128)
    assert from_bad.sum() >= 15 and kept.tolist() == [130]
    k, v, _ = gqa.views(after, 2, dim)
    for c in range(3):
        page, at = int(to[0, c]), from_bad[64 * c:64 * c + 64]
        there = mine[64 * c:64 * c + 64] >= 0
        for codes in (k[page, 1], v[page, 1].T):
            assert torch.equal(torch.isnan(gqa.value_of(codes)).all(-1)[there], at[there])
            assert torch.isfinite(gqa.value_of(codes))[there & ~at].all()
    q, cu = _gqa.queries(1, 8, dim, 183), torch.tensor([0, 1], dtype=I32)
    for p, tab, n in ((pages, table, lens), (after, to, kept)):
        out, lse = run(cuda, q, p, tab, cu, n, 2)
        check(cuda, q, p, tab, cu, n, 2, out, lse)
        assert torch.isnan(out[:, 4:]).all() and torch.isnan(lse[:, 4:]).all() and torch.isfinite(out[:, :4]).all()
        got = torch.zeros(pages.shape[0], 2, 64, device=cuda)
        finite = torch.nan_to_num(lse, nan=1.0)
        gqa_cache_weights(*_gqa.to(cuda, q), finite, *_gqa.to(cuda, p, tab, cu, n), got)
        check_sums(cuda, q, finite, p, tab, cu, n, 2, torch.zeros(got.shape), got, True)
