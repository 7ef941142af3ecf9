"""flash_paged_mla where the weights of a row's keys, or the keys' scales, are far apart: one key that has most of a row's
weight before a long flat tail, keys of very different sizes in one page, keys that a row does not see.

The tolerance is that of test_gpu_flash_paged_mla (bf16's half step of the result, 2^-8 of it; as much of
sum_j p_j |latent_j| for the weights; the scores' error) and what a weight much smaller than another one of the same
32 keys loses.  x = p_j scale_j over the power of two that brings the largest of the 32 into [128, 256) is held as two e4m3
numbers, hi + lo / 32, whose smallest steps are 2^-9 and 2^-9 / 32 = 2^-14: where x is too small for 2^-8 of it, it is off by
half of the latter, 2^-15, at most, which is 2^-22 of the largest, 128 or more.  An output's sum of |code| times that, over
the keys of each 32, is the term `beside`.  An exponential below 2^-126 of the row's largest is below fp32's normal numbers and
may be 0: 2^-126 of sum_j |latent_j| over the keys.

Every number of tokens per sequence runs in its own tile height (16, 32 and 64 rows)."""
import math

import pytest
import torch

from oracle import paged
from tests import _paged
from tests.test_gpu_flash_paged_mla import SCALE, queries, run
from tilert_amd.flash_paged_mla import flash_paged_mla

pytestmark = pytest.mark.gpu
BF16, FP8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


def put(pages, ids, latent, rope):
    """Keys 0 .. n - 1 into the pages `ids` (all on the GPU), quantised per key; latent [n, 512], rope [n, 64] fp32."""
    codes, scales, ropes = paged.views(pages)
    p = torch.arange(latent.shape[0], device=latent.device)
    at = (ids[p // 64].long(), p % 64)
    s = latent.abs().amax(-1).clamp_min(1e-4) / 448
    codes.view(torch.uint8)[at] = (latent / s[:, None]).clamp(-448, 448).to(FP8).view(torch.uint8)
    scales[at] = s
    ropes[at] = rope.to(BF16)


def definition(q, qp, pages, ids, n, scale, cut=False):
    """(out, lse, tolerance of out, of lse) in fp64 for one token, q [heads, 512], that sees the first n keys of `ids`.
    `cut`: with the most that the fp8 MFMA's sums are off where a few dims' products are far above the others'.  It adds
    eight consecutive dims' products at a time, aligned to the largest and cut 13 bits below it: up to 7 of them lose
    2^-13 of the largest each, and as much of the second half of the query, which is 2^-4 of it at most: 7 x 17 / 16 < 7.5."""
    codes, scales, rope = paged.views(pages)
    p = torch.arange(n, device=q.device)
    at = (ids[p // 64].long(), p % 64)
    code, s = codes.view(torch.uint8)[at].view(FP8).double(), scales[at].double()
    latent, pe = code * s[:, None], rope[at].double()
    z = (q.double() @ latent.T + qp.double() @ pe.T) * scale
    size = (q.double().abs() @ latent.abs().T + qp.double().abs() @ pe.abs().T) * scale
    lse = torch.logsumexp(z, -1)
    w = torch.exp(z - lse[:, None])
    slack = size.max(-1).values * 600 * 2.0 ** -24 + n * 2.0 ** -24
    if cut:
        largest = (q.double().abs()[:, None] * latent.abs()).view(q.shape[0], n, 64, 8).amax(-1).sum(-1)
        slack = slack + 7.5 * 2.0 ** -13 * scale * largest.max(-1).values
    pad = -n % 32
    top = torch.nn.functional.pad(w * s, (0, pad)).view(w.shape[0], -1, 32).amax(-1)
    beside = 2.0 ** -22 * top @ torch.nn.functional.pad(code.abs(), (0, 0, 0, pad)).view(-1, 32, 512).sum(1)
    out = w @ latent
    tol = 2 ** -8 * out.abs() + (2 ** -8 + 2 * (slack[:, None] + 2 ** -18)) * (w @ latent.abs()) + beside + 2.0 ** -126 * latent.abs().sum(0)
    return out, lse, tol, slack + 2 ** -20 * (1 + lse.abs())


def close(out, lse, q, qp, pages, ids, first, tokens, scale=SCALE, cut=False):
    """The tokens' results against the definition's; the sequence's first token is at position `first`."""
    for t in tokens:
        want, want_lse, tol, tol_lse = definition(q[t], qp[t], pages, ids, first + t + 1, scale, cut)
        off = (out[t].double() - want).abs()
        assert torch.all(off <= tol), (t, (off / tol).max())
        assert torch.all((lse[t].double() - want_lse).abs() <= tol_lse), t


def check_all(case, out, lse, scale=SCALE, cut=False):
    new = case[0].shape[0]
    close(out, lse, case[0], case[1], case[2], case[3][0], int(case[5][0]) - new, range(new), scale, cut)


def sink_case(cuda, keys, mass, mean, seed):
    """One key with `mass` of a row's weight, the others' scores within about 0.4 of each other."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    n = -(-keys // 64)
    pages = torch.empty(n, paged.PAGE_BYTES, dtype=torch.uint8, device=cuda)
    ids = torch.randperm(n, generator=g, device=cuda).to(I32)
    rope = torch.randn(keys, 64, generator=g, device=cuda) * 0.05
    # 64 x 0.5 x c x SCALE over the tail's scores of mean 0
    rope[0] = math.log(mass / (1 - mass) * keys) / (64 * 0.5 * SCALE)
    latent = torch.randn(keys, 512, generator=g, device=cuda) + mean * torch.randn(512, generator=g, device=cuda)
    put(pages, ids, latent, rope)
    return g, pages, ids


def sink_queries(cuda, g, tokens, heads):
    q = (torch.randn(tokens, heads, 512, generator=g, device=cuda) * 0.1).to(BF16)
    return q, torch.full((tokens, heads, 64), 0.5, dtype=BF16, device=cuda)


@pytest.mark.parametrize("tokens,keys,mass,mean", [
    (1024, 16384, 0.9, 0.0), (1024, 16384, 0.97, 1.0), (1024, 32768, 0.97, 0.0), (1024, 65536, 0.5, 1.0),
    (1024, 131072, 0.9, 0.0), (8320, 9000, 0.9, 1.0),  # the last: more tiles than are split
])
def test_a_long_tail_behind_one_heavy_key(cuda, tokens, keys, mass, mean):
    """Each workgroup walks a whole cache, or half of one, in 64-row tiles."""
    g, pages, ids = sink_case(cuda, keys, mass, mean, tokens + keys)
    q, qp = sink_queries(cuda, g, tokens, 16)
    out, lse = torch.empty_like(q), torch.empty(tokens, 16, device=cuda)
    cu, lens = torch.tensor([0, tokens], dtype=I32, device=cuda), torch.tensor([keys], dtype=I32, device=cuda)
    flash_paged_mla(q, qp, pages, ids[None], cu, lens, out, lse, model_arch="deepseek_v3_2")
    some = [0, 1, tokens // 2, tokens - 3, tokens - 1]
    close(out, lse, q, qp, pages, ids, keys - tokens, some)


@pytest.mark.parametrize("heads", [16, 32])
@pytest.mark.parametrize("keys,mass,mean", [(16384, 0.9, 0.0), (32768, 0.97, 1.0)])
def test_a_long_tail_in_a_decode_batch(cuda, heads, keys, mass, mean):
    """256 sequences over the same pages, so that each has about one workgroup, in 16-row and 32-row tiles."""
    g, pages, ids = sink_case(cuda, keys, mass, mean, heads + keys)
    q, qp = sink_queries(cuda, g, 256, heads)
    out, lse = torch.empty_like(q), torch.empty(256, heads, device=cuda)
    cu, lens = torch.arange(257, dtype=I32, device=cuda), torch.full((256,), keys, dtype=I32, device=cuda)
    flash_paged_mla(q, qp, pages, ids.expand(256, -1).contiguous(), cu, lens, out, lse, model_arch="deepseek_v3_2")
    for t in (0, 100, 255):
        close(out[t:t + 1], lse[t:t + 1], q[t:t + 1], qp[t:t + 1], pages, ids, keys - 1, [0])


TILES = [(1, 16), (2, 16), (1, 64), (24, 16)]  # new tokens, heads: 16, 32, 32 and 64 rows a tile


def _sized(cuda, new, total, heads, seed):
    """(q, qp, pages, table, cu, lens, scales view) on the GPU; queries have no part in dims 256 and up, where a key may then
    hold anything without a score of it."""
    pages, table, cu, lens, rows = _paged.batch([new], [total], seed=seed)
    _paged.fill(pages, table, [total], seed=seed)
    q, qp = queries(rows, heads, seed)
    q[..., 256:] = 0
    return _paged.to(cuda, q, qp, pages, table, cu, lens)


def _enlarge(case, key, factor, rope=None):
    """The key's latent moved to dims 256 and up, `factor` times as large."""
    codes, scales, ropes = paged.views(case[2])
    page, row = int(case[3][0, key // 64]), key % 64
    codes.view(torch.uint8)[page, row, :256] = 0
    scales[page, row] *= factor
    if rope is not None:
        ropes[page, row] = rope


@pytest.mark.parametrize("power", [4, 10, 12, 14, 20, 60, 110])
@pytest.mark.parametrize("new,total", [(8, 200), (24, 64), (24, 1000)])
def test_a_large_key_that_a_row_does_not_see(cuda, new, total, power):
    """The last token's key, times 2^power: every earlier token's result is the same bit for bit."""
    case = _sized(cuda, new, total, 16, 101)
    before = run(cuda, *case)
    _enlarge(case, total - 1, 2.0 ** power)
    after = run(cuda, *case)
    assert torch.equal(before[0][:-1], after[0][:-1]) and torch.equal(before[1][:-1], after[1][:-1])
    check_all(case, *after)


@pytest.mark.parametrize("power", [10, 20, 60])
@pytest.mark.parametrize("new,heads", TILES)
@pytest.mark.parametrize("total,at", [(300, 0), (300, 130), (900, 3), (900, 800)])
def test_a_large_key_of_no_weight(cuda, new, heads, total, at, power):
    """A key that all rows see, 2^power times the others, with a weight of less than e^-100 of theirs."""
    case = _sized(cuda, new, total, heads, 103)
    case[1].fill_(0.5)
    _enlarge(case, at, 2.0 ** power, rope=-30.0)  # a score of 64 x 0.5 x -30 x SCALE = -130
    check_all(case, *run(cuda, *case))


@pytest.mark.parametrize("powers", [8, 16, 24])
@pytest.mark.parametrize("new,heads", TILES)
@pytest.mark.parametrize("total", [100, 700, 3000])
def test_keys_of_very_different_sizes(cuda, new, heads, total, powers):
    """Scales spread over 2^0 .. 2^powers inside each page, weights all of one order: queries without a latent part."""
    case = _sized(cuda, new, total, heads, 107)
    case[0].zero_()
    g = torch.Generator().manual_seed(109)
    scales = paged.views(case[2])[1]
    scales *= torch.pow(2.0, torch.randint(0, powers + 1, scales.shape, generator=g).float()).to(cuda)
    check_all(case, *run(cuda, *case))


@pytest.mark.parametrize("new,heads", TILES)
@pytest.mark.parametrize("first", [0, 64, 256])
def test_keys_of_scale_zero_with_all_the_weight(cuda, new, heads, first):
    """Keys without a latent, from page `first` / 64 on, whose rope parts outweigh the others' by e^200: zeros, and the lse."""
    total = first + 100
    case = _sized(cuda, new, total, heads, 113)
    case[1].fill_(0.5)
    codes, scales, ropes = paged.views(case[2])
    p = torch.arange(first, total - new, device=cuda)
    at = (case[3][0, p // 64].long(), p % 64)
    codes.view(torch.uint8)[at], scales[at], ropes[at] = 0, 0.0, 46.0
    out, lse = run(cuda, *case)
    check_all(case, out, lse)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
