"""add_rmsnorm_quant on rows that hold a NaN or an infinity: the quantised outputs show it as the definition does, also where
the bf16 output is left out, and codes are finite whatever a row held."""
import pytest
import torch

from oracle import paged
from tests.test_gpu_add_rmsnorm_quant import E, LOGS, _inputs, _outs
from tilert_amd.rmsnorm import add_rmsnorm_quant

pytestmark = pytest.mark.gpu
KW = {"model_arch": "deepseek_v3_2"}


@pytest.mark.parametrize("fmt", ["div", None, "ue8m0"])
@pytest.mark.parametrize("dim", [128, 1536, 7168, 10240])
@pytest.mark.parametrize("with_y", [True, False])
def test_scales_show_a_bad_row(cuda, dim, fmt, with_y):
    x, r, gamma = _inputs(6, dim, dim, cuda)
    clean, bad = _outs(x), _outs(x)
    add_rmsnorm_quant(x, r, gamma, *clean, LOGS, scale_fmt=fmt, **KW)
    x[1, dim // 2], r[2, dim - 1], x[3, 0] = float("nan"), float("inf"), -float("inf")
    x[4, 1], r[4, 1] = float("inf"), -float("inf")
    add_rmsnorm_quant(x, r, gamma, bad[0], bad[1] if with_y else None, bad[2], bad[3], LOGS, scale_fmt=fmt, **KW)
    q, s = bad[2], bad[3]
    n = paged.norm(x.double() + r.double(), gamma, 1e-6)  # a NaN anywhere: all NaN; an infinity: NaN there, 0 elsewhere
    want_bad = ~torch.isfinite(n.view(6, -1, 128)).all(-1)
    assert torch.equal(torch.isnan(s), want_bad)
    assert want_bad[1].all() and want_bad[4].all() and int(want_bad[2].sum()) == 1 and int(want_bad[3].sum()) == 1
    assert torch.isfinite(q.float()).all()
    back = (q.float().view(6, -1, 128) * s[..., None]).view(6, dim)
    assert torch.equal(torch.isnan(back.view(6, -1, 128)).all(-1), want_bad)
    assert torch.all(back[2:4][(n[2:4] == 0) & ~want_bad[2:4].repeat_interleave(128, 1)] == 0)
    for row in (0, 5):
        assert torch.equal(s[row], clean[3][row]) and torch.equal(q[row].view(torch.uint8), clean[2][row].view(torch.uint8))


@pytest.mark.parametrize("fmt", ["div", None, "ue8m0"])
def test_a_gamma_that_is_not_finite_is_its_group_s(cuda, fmt):
    x, r, gamma = _inputs(4, 1024, 9, cuda)
    clean, bad = _outs(x), _outs(x)
    add_rmsnorm_quant(x, r, gamma, *clean, LOGS, scale_fmt=fmt, **KW)
    gamma[300], gamma[900] = float("nan"), float("inf")
    x[0, 300] = r[0, 300] = 0  # 0 * NaN, and a finite element times an infinite gamma
    add_rmsnorm_quant(x, r, gamma, *bad, LOGS, scale_fmt=fmt, **KW)
    groups = torch.zeros(8, dtype=torch.bool, device=cuda)
    groups[2] = groups[7] = True
    assert torch.isnan(bad[3][:, groups]).all() and torch.isfinite(bad[3][:, ~groups]).all()
    assert torch.isfinite(bad[2].float()).all()
    assert torch.equal(bad[3][1:, ~groups], clean[3][1:, ~groups])
