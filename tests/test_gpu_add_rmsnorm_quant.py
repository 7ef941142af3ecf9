"""GPU parity of add_rmsnorm_quant against its definition in 64 bits.

Tolerances: fp32 sums over a row of d columns in chains of at most d / 2048 * 8 + 25 roundings, halved by the root, and
six more operations: below 2^-18 of a norm value.  Half a step of bf16 is 2^-8 of the value, of e4m3 2^-4 (2^-10 of the
scale below the normal range)."""
import pytest
import torch

from oracle import paged
from tilert_amd.rmsnorm import add_rmsnorm_quant

pytestmark = pytest.mark.gpu
LOGS = torch.zeros(1)
E = 2.0 ** -18


def _inputs(rows, dim, seed, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, dim, generator=g).to(torch.bfloat16)
    r = (torch.randn(rows, dim, generator=g) * 3).to(torch.bfloat16)
    x[0, :128] = 0.0
    r[0, :128] = 0.0  # a group of zeros
    return x.to(dev), r.to(dev), (torch.rand(dim, generator=g) + 0.5).to(dev)


def _outs(x):
    return (torch.empty_like(x), torch.empty_like(x), torch.empty_like(x, dtype=torch.float8_e4m3fn),
            torch.empty(*x.shape[:-1], x.shape[-1] // 128, device=x.device))


@pytest.mark.parametrize("rows,dim,fmt", [(1, 128, "div"), (4, 7168, None), (1, 7168, "div"), (7, 6144, "div"),
                                          (3, 2048, "ue8m0"), (5, 2176, None), (2, 8192, "div"), (3, 8320, "div"),
                                          (33, 16384, None), (300, 7168, "div"), (1030, 1536, "div"), (2500, 1664, "div"),
                                          (700, 10240, "div"), (0, 7168, "div")])
def test_against_64_bits(cuda, rows, dim, fmt):
    if rows == 0:
        x, r, gamma = (torch.empty(0, dim, dtype=torch.bfloat16, device=cuda) for _ in range(2)), None, None
        x, r = x
        gamma = torch.ones(dim, device=cuda)
    else:
        x, r, gamma = _inputs(rows, dim, rows + dim, cuda)
    out, y, q, s = _outs(x)
    add_rmsnorm_quant(x, r, gamma, out, y, q, s, LOGS, model_arch="deepseek_v3_2", scale_fmt=fmt)
    if rows == 0:
        return
    assert torch.equal(out, (x.float() + r.float()).to(torch.bfloat16))  # an fp32 sum of two bf16 values, rounded once
    n = paged.norm(x.double() + r.double(), gamma, 1e-6)
    assert torch.all((y.double() - n).abs() <= (2 ** -8 + E) * n.abs())
    want_s = paged.scale_of(n.view(rows, -1, 128).abs().amax(-1), fmt)
    if fmt == "ue8m0":  # a power of two; a largest value within rounding of 448 s may fall on either side
        ratio = s.double() / want_s
        assert torch.all((ratio == 1) | (ratio == 2) | (ratio == 0.5)) and (ratio == 1).double().mean() > 0.99
    else:
        assert torch.all((s.double() - want_s).abs() <= 2 * E * want_s)
    wide = s.double().repeat_interleave(128, 1)
    off = (q.double() * wide - n).abs()
    assert torch.all(off <= torch.maximum(2 ** -4 * n.abs(), 2 ** -10 * wide) + 2 * E * n.abs())


@pytest.mark.parametrize("rows,dim", [(4, 7168), (600, 2048)])
def test_in_place_and_left_out_outputs(cuda, rows, dim):
    x, r, gamma = _inputs(rows, dim, 3, cuda)
    out, y, q, s = _outs(x)
    kw = {"model_arch": "deepseek_v3_2", "scale_fmt": "div"}
    add_rmsnorm_quant(x, r, gamma, out, y, q, s, LOGS, **kw)
    for alias in (x, r):
        a, b = x.clone(), r.clone()
        target = a if alias is x else b
        y2, q2, s2 = (torch.zeros_like(t) for t in (y, q, s))
        add_rmsnorm_quant(a, b, gamma, target, y2, q2, s2, LOGS, **kw)
        assert torch.equal(target, out) and torch.equal(y, y2) and torch.equal(s, s2)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8))
    y3, q3, s3, o3 = torch.zeros_like(y), torch.zeros_like(q), torch.zeros_like(s), torch.zeros_like(out)
    add_rmsnorm_quant(x, r, gamma, o3, y3, profile_logs=LOGS, **kw)
    assert torch.equal(y3, y) and torch.equal(o3, out)
    add_rmsnorm_quant(x, r, gamma, o3, None, q3, s3, LOGS, **kw)
    assert torch.equal(q3.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s3, s)


def test_a_bad_row_touches_no_other(cuda):
    x, r, gamma = _inputs(6, 7168, 5, cuda)
    kw = {"model_arch": "deepseek_v3_2", "scale_fmt": "div"}
    clean, bad = _outs(x), _outs(x)
    add_rmsnorm_quant(x, r, gamma, *clean, LOGS, **kw)
    x[2, 100], r[4, 7000] = float("nan"), float("inf")
    add_rmsnorm_quant(x, r, gamma, *bad, LOGS, **kw)
    keep = [0, 1, 3, 5]
    for a, b in zip(clean, bad):
        assert torch.equal(a.view(torch.uint8)[keep] if a.element_size() == 1 else a[keep],
                           b.view(torch.uint8)[keep] if b.element_size() == 1 else b[keep])
    assert torch.isnan(bad[1][2]).all() and torch.isnan(bad[1][4]).any()


def test_bf16_gamma_is_widened(cuda):
    x, r, gamma = _inputs(2, 256, 7, cuda)
    kw = {"model_arch": "deepseek_v3_2"}
    a, b = _outs(x), _outs(x)
    add_rmsnorm_quant(x, r, gamma.to(torch.bfloat16), *a, LOGS, **kw)
    add_rmsnorm_quant(x, r, gamma.to(torch.bfloat16).float(), *b, LOGS, **kw)
    assert torch.equal(a[1], b[1])
