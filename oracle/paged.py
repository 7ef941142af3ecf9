"""The paged latent cache's operators and the residual norm in 64 bits, sequence by sequence, from their definitions.

Pages are uint8 [n_pages, 41216]: 64 keys x 512 e4m3fn codes, 64 fp32 scales, 64 x 64 bf16 rope parts.  A batch is
(block_table, cu_seqlens, seq_lens) as lists or tensors; a key named by no valid page is not there.
"""
from __future__ import annotations

import math

import torch

PAGE_BYTES, KEYS, LATENT, ROPE = 41216, 64, 512, 64
_SCALE_AT, _ROPE_AT = KEYS * LATENT, KEYS * LATENT + KEYS * 4


def views(pages: torch.Tensor):
    """(codes e4m3fn [n, 64, 512], scales fp32 [n, 64], rope bf16 [n, 64, 64]) as views of the pages."""
    n = pages.shape[0]
    return (pages[:, :_SCALE_AT].view(n, KEYS, LATENT).view(torch.float8_e4m3fn),
            pages[:, _SCALE_AT:_ROPE_AT].view(torch.float32), pages[:, _ROPE_AT:].view(torch.bfloat16).view(n, KEYS, ROPE))


def places(n_pages: int, table: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor, rows: int):
    """(token, page, row) of every token of the batch that has a place."""
    out = []
    table, cu, lens = table.tolist(), cu.tolist(), lens.tolist()
    for b, L in enumerate(lens):
        for t in range(cu[b], min(cu[b + 1], rows)):
            pos = L - cu[b + 1] + t
            if 0 <= pos < len(table[b]) * KEYS and 0 <= table[b][pos // KEYS] < n_pages:
                out.append((t, table[b][pos // KEYS], pos % KEYS))
    return out


def scale_of(amax: torch.Tensor, scale_fmt) -> torch.Tensor:
    """The act_quant scale of a group's largest magnitude (fp64 in and out; the power of two of "ue8m0" exactly)."""
    amax = amax.clamp_min(1e-4)
    if scale_fmt == "ue8m0":
        return torch.pow(2.0, torch.ceil(torch.log2(amax / 448)))
    return amax / 448


def norm(x: torch.Tensor, gamma, eps: float) -> torch.Tensor:
    x = x.double()
    if gamma is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()


def rope(pe: torch.Tensor, freqs, interleaved: bool) -> torch.Tensor:
    z = pe.double()
    if freqs is None:
        return z
    w = freqs.double().reshape(-1, ROPE // 2, 2)
    a, b = (z[:, 0::2], z[:, 1::2]) if interleaved else (z[:, :32], z[:, 32:])
    out = torch.empty_like(z)
    lo, hi = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, 32), slice(32, 64))
    out[:, lo] = a * w[..., 0] - b * w[..., 1]
    out[:, hi] = a * w[..., 1] + b * w[..., 0]
    return out


def attention(q, q_pe, pages, table, cu, lens, scale: float):
    """(out, lse, spread, slack) in fp64 for every row; rows of no sequence are NaN.  spread = sum_j p_j |latent_j| and
    slack = the bound of a score's error when its 576 products are summed in fp32, for a test's tolerance."""
    codes, scales, rope_k = views(pages)
    T, H = q.shape[0], q.shape[1]
    dev = q.device
    out = torch.full((T, H, LATENT), math.nan, dtype=torch.float64, device=dev)
    lse, spread, slack = out[..., 0].clone(), out.clone(), out[..., 0].clone()
    for b, L in enumerate(lens.tolist()):
        c0, c1 = int(cu[b]), min(int(cu[b + 1]), T)
        base = L - int(cu[b + 1])
        n = max(0, min(L, table.shape[1] * KEYS))
        p = torch.arange(n, device=dev)
        page = table[b].to(dev)[p // KEYS].long()
        p, page = p[(page >= 0) & (page < pages.shape[0])], page[(page >= 0) & (page < pages.shape[0])]
        at = (page, p % KEYS)
        latent = codes.view(torch.uint8)[at].view(torch.float8_e4m3fn).double() * scales[at].double()[:, None]
        pe = rope_k[at].double()
        for t in range(c0, c1):
            k = int((p <= base + t).sum())
            if k == 0:
                out[t], lse[t], spread[t], slack[t] = 0, -math.inf, 0, 0
                continue
            z = (q[t].double() @ latent[:k].T + q_pe[t].double() @ pe[:k].T) * scale
            size = (q[t].double().abs() @ latent[:k].abs().T + q_pe[t].double().abs() @ pe[:k].abs().T) * scale
            lse[t] = torch.logsumexp(z, -1)
            w = torch.exp(z - lse[t][:, None])
            out[t], spread[t] = w @ latent[:k], w @ latent[:k].abs()
            slack[t] = size.max(-1).values * 600 * 2.0 ** -24 + k * 2.0 ** -24
    return out, lse, spread, slack
