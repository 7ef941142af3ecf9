"""GPU parity of the paged latent cache's writer and reader against their definitions in 64 bits.

Tolerances.  The norm in fp32: a sum of 512 squares in a tree (14 roundings), one division, root, reciprocal and two
products, each at most 2^-24 relative: below 2^-19 in n and in the scale.  A code is off by half a step: 2^-4 of the
value, or 2^-10 of the scale below the normal range.  bf16: 2^-8 of the value."""
import math

import pytest
import torch

from oracle import paged
from tests import _paged
from tilert_amd.mla_cache import KV_PAGE_BYTES, mla_cache_read, mla_cache_write

pytestmark = pytest.mark.gpu
E = 2.0 ** -19


def _inputs(rows, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    kv = (torch.randn(rows, 512, generator=g) * std).to(torch.bfloat16)
    pe = torch.randn(rows, 64, generator=g).to(torch.bfloat16)
    gamma = torch.rand(512, generator=g) * 0.2 + 0.9
    angle = torch.rand(rows, 32, generator=g, dtype=torch.float64) * 2 * math.pi
    return kv, pe, gamma, torch.stack([angle.cos(), angle.sin()], -1).float().reshape(rows, 1, 64)


BATCHES = [
    ([1], [1], 0), ([1], [64], 0), ([1], [65], 2), ([5], [5], 0),
    ([4, 1, 0, 130, 3], [100, 1, 77, 130, 66], 3),
    ([1] * 70, list(range(1, 71)), 0),              # more sequences than a wave has lanes
    ([0, 2, 0, 0, 7], [0, 64, 3, 0, 200], 1),       # empty sequences, one of no keys
]


@pytest.mark.parametrize("new,total,pad", BATCHES)
@pytest.mark.parametrize("fmt,normed,turned,interleaved", [("div", True, True, True), (None, False, True, False),
                                                         ("ue8m0", True, False, True)])
def test_write(cuda, new, total, pad, fmt, normed, turned, interleaved):
    pages, table, cu, lens, rows = _paged.batch(new, total, pad=pad, seed=3)
    kv, pe, gamma, freqs = _inputs(rows, 5)
    if rows > 1:
        kv[1] = 0  # a key of zeros
    gamma, freqs = gamma if normed else None, freqs if turned else None
    got = pages.to(cuda)
    d = _paged.to(cuda, kv, pe, table, cu, lens, gamma, freqs)
    mla_cache_write(d[0], d[1], got, d[2], d[3], d[4], d[5], d[6], scale_fmt=fmt, interleaved=interleaved)
    got = got.cpu()
    n, z = paged.norm(kv, gamma, 1e-6), paged.rope(pe, freqs, interleaved)
    s = paged.scale_of(n.abs().amax(-1), fmt)
    codes, scales, rope = paged.views(got)
    size = pe.double().abs().max() * 2
    written = torch.zeros(got.shape[0], 64, dtype=torch.bool)
    for t, page, row in paged.places(got.shape[0], table, cu, lens, rows):
        written[page, row] = True
        sc = scales[page, row].double()
        assert (sc - s[t]).abs() <= E * s[t]
        value = codes[page, row].double() * sc
        assert torch.all((value - n[t]).abs() <= torch.maximum(2 ** -4 * n[t].abs(), 2 ** -10 * sc) + 2 * E * n[t].abs())
        off = (rope[page, row].double() - z[t]).abs()
        assert torch.all(off <= 2 ** -8 * z[t].abs() + (2 ** -22 * size if turned else 0))
    blank = got.view(torch.uint8)[:, :64 * 512].view(-1, 64, 512)[~written]
    assert torch.all(blank == 0xff) and torch.all(rope.view(torch.int16)[~written] == -1)
    assert torch.all(scales.view(torch.int32)[~written] == -1)


@pytest.mark.parametrize("new,total,pad", BATCHES)
def test_read(cuda, new, total, pad):
    pages, table, cu, lens, rows = _paged.batch(new, total, pad=pad, seed=7)
    _paged.fill(pages, table, total)
    kv = torch.full((rows, 512), 7.0, dtype=torch.bfloat16, device=cuda)
    pe = torch.full((rows, 64), 7.0, dtype=torch.bfloat16, device=cuda)
    mla_cache_read(*_paged.to(cuda, pages, table, cu, lens), kv, pe)
    codes, scales, rope = paged.views(pages)
    want_kv, want_pe = torch.full((rows, 512), 7.0, dtype=torch.bfloat16), torch.full((rows, 64), 7.0, dtype=torch.bfloat16)
    for t, page, row in paged.places(pages.shape[0], table, cu, lens, rows):
        want_kv[t] = (codes[page, row].float() * scales[page, row]).to(torch.bfloat16)  # one product, one rounding
        want_pe[t] = rope[page, row]
    assert torch.equal(kv.cpu(), want_kv) and torch.equal(pe.cpu(), want_pe)


def test_rows_without_a_place(cuda):
    """Positions below 0 or past the table, and pages outside the pool: nothing is written for them, nothing read."""
    pages, table, cu, lens, rows = _paged.batch([70, 6, 5], [130, 6, 5], seed=9)
    _paged.fill(pages, table, [130, 6, 5])
    table[0, 1] = pages.shape[0]   # page outside the pool
    table[2, 0] = -5
    lens[0] = 70 + 150             # positions 150 .. 219: past the table's 192
    lens[1] = 4                    # positions -2 .. 3
    kv, pe, _, _ = _inputs(rows, 11)
    got = pages.to(cuda)
    d = _paged.to(cuda, kv, pe, table, cu, lens)
    mla_cache_write(d[0], d[1], got, *d[2:])
    want_rows = {(page, row): t for t, page, row in paged.places(pages.shape[0], table, cu, lens, rows)}
    before, after = paged.views(pages)[2], paged.views(got.cpu())[2]
    for page in range(pages.shape[0]):
        for row in range(64):
            t = want_rows.get((page, row))
            want = before[page, row] if t is None else pe[t]
            assert torch.equal(after[page, row].view(torch.int16), want.view(torch.int16)), (page, row, t)
    out, out_pe = torch.full_like(d[0], 3.0), torch.full_like(d[1], 3.0)
    mla_cache_read(got, *d[2:], out, out_pe)
    there = torch.zeros(rows, dtype=torch.bool)
    there[list(want_rows.values())] = True
    assert torch.all(out.cpu()[~there] == 3.0) and torch.equal(out_pe.cpu()[there], pe[there])


def test_keys_with_nan_or_infinity_read_back_as_nan(cuda):
    pages, table, cu, lens, rows = _paged.batch([4], [4], seed=13)
    kv, pe, gamma, _ = _inputs(rows, 15)
    kv[1, 77], kv[2, 500] = math.nan, math.inf
    for g in (None, gamma.to(cuda)):
        got = pages.to(cuda)
        d = _paged.to(cuda, kv, pe, table, cu, lens)
        mla_cache_write(d[0], d[1], got, *d[2:], g)
        out, out_pe = torch.zeros_like(d[0]), torch.zeros_like(d[1])
        mla_cache_read(got, *d[2:], out, out_pe)
        assert torch.isnan(out[1:3]).all() and torch.isfinite(out[[0, 3]]).all()
        codes = paged.views(got.cpu())[0].float()
        assert torch.isfinite(codes[int(table[0, 0]), :4]).all()  # no code is NaN, whatever was written


def test_large_and_tiny_keys(cuda):
    """The largest bf16 values and ones below the scale's floor quantise and read back within half a step."""
    pages, table, cu, lens, rows = _paged.batch([3], [3], seed=17)
    kv, pe, _, _ = _inputs(rows, 19)
    kv[0] *= 1e38 / kv[0].abs().max()
    kv[1] *= 1e-30
    kv[2] = torch.finfo(torch.bfloat16).max
    got = pages.to(cuda)
    d = _paged.to(cuda, kv, pe, table, cu, lens)
    mla_cache_write(d[0], d[1], got, *d[2:])
    out, out_pe = torch.zeros_like(d[0]), torch.zeros_like(d[1])
    mla_cache_read(got, *d[2:], out, out_pe)
    x, y = kv.double(), out.cpu().double()
    s = paged.scale_of(x.abs().amax(-1), "div")
    assert torch.isfinite(y).all()
    assert torch.all((y - x).abs() <= torch.maximum(2 ** -4 * x.abs(), 2 ** -10 * s[:, None]) * (1 + 2 ** -7))


def test_page_size():
    assert KV_PAGE_BYTES == paged.PAGE_BYTES
