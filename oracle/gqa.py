"""The paged per-head cache's operators in 64 bits, sequence by sequence and head by head, from their definitions.

Pages are uint8 [n_pages, kv * 128 * dim + scales padded to 128]: for each kv head 64 x dim e4m3fn key codes, then dim x 64
value codes; behind all heads fp32 scales [kv, 2].  A batch is (block_table, cu_seqlens, seq_lens); a key named by no valid
page is not there.
"""
from __future__ import annotations

import math

import torch

KEYS = 64
F32, F64, FP8, U8 = torch.float32, torch.float64, torch.float8_e4m3fn, torch.uint8


def page_bytes(kv: int, dim: int) -> int:
    return kv * 128 * dim + -(-kv * 8 // 128) * 128


def views(pages: torch.Tensor, kv: int, dim: int):
    """(key codes u8 [n, kv, 64, dim], value codes u8 [n, kv, dim, 64], scales fp32 [n, kv, 2]) as views of the pages."""
    n, codes = pages.shape[0], kv * 128 * dim
    both = pages[:, :codes].view(n, kv, 2, KEYS * dim)
    return (both[:, :, 0].view(n, kv, KEYS, dim), both[:, :, 1].view(n, kv, dim, KEYS),
            pages[:, codes:codes + kv * 8].view(F32).view(n, kv, 2))


def scale_of(amax: float) -> float:
    """The least power of two s with max(amax, 1e-4) <= 448 s."""
    mantissa, exponent = math.frexp(max(amax, 1e-4))
    return math.ldexp(1.0, exponent - 9 + (mantissa > 0.875))


def value_of(codes: torch.Tensor) -> torch.Tensor:
    return codes.contiguous().view(FP8).double()


def turned(x, gamma, freqs, interleaved: bool, eps: float) -> torch.Tensor:
    """[tokens, heads, dim]: each row's RMSNorm, its first dims turned by the token's freqs [tokens, rope]."""
    x = x.double()
    if gamma is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * gamma.double()
    if freqs is None:
        return x
    w = freqs.double().reshape(x.shape[0], 1, -1, 2)
    r = w.shape[2] * 2
    out = x.clone()
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    out[..., lo] = x[..., lo] * w[..., 0] - x[..., hi] * w[..., 1]
    out[..., hi] = x[..., lo] * w[..., 1] + x[..., hi] * w[..., 0]
    return out


def keys_of(pages, table, b: int, n: int, kv: int, dim: int):
    """Positions below n of sequence b that are there, and their keys and values [kv, keys, dim]."""
    k, v, scales = views(pages, kv, dim)
    p = torch.arange(max(0, min(n, table.shape[1] * KEYS)), device=pages.device)
    page = table[b].to(pages.device)[p // KEYS].long()
    fine = (page >= 0) & (page < pages.shape[0])
    p, page = p[fine], page[fine]
    s = scales[page].double().permute(2, 1, 0)[..., None]
    s = torch.where((s > 0) & torch.isfinite(s), s, math.nan)
    s = torch.where(torch.isnan(s).any(0), math.nan, s)  # (one of a block's two that is no scale: its keys are NaN)
    return p, value_of(k[page, :, p % KEYS]).transpose(0, 1) * s[0], value_of(v[page, :, :, p % KEYS]).transpose(0, 1) * s[1]


def attention(q, pages, table, cu, lens, kv: int, scale: float):
    """(out, lse, spread, slack) in fp64 for every row; rows of no sequence are NaN.  spread = sum_j p_j |v_j| and slack = the
    bound of a score's error when its products are summed in fp32 and the score rounded on its way to the exponent."""
    T, H, D = q.shape
    out = torch.full((T, H, D), math.nan, dtype=F64, device=q.device)
    lse, spread, slack = out[..., 0].clone(), out.clone(), out[..., 0].clone()
    G = H // kv
    for b, L in enumerate(lens.tolist()):
        c0, c1 = int(cu[b]), min(int(cu[b + 1]), T)
        base = L - int(cu[b + 1])
        p, k, v = keys_of(pages, table, b, L, kv, D)
        for t in range(c0, c1):
            n = int((p <= base + t).sum())
            if n == 0:
                out[t], lse[t], spread[t], slack[t] = 0, -math.inf, 0, 0
                continue
            x = q[t].double().view(kv, G, D)
            z = (x @ k[:, :n].transpose(1, 2)).view(H, n) * scale
            size = (x.abs() @ k[:, :n].abs().transpose(1, 2)).view(H, n) * scale
            lse[t] = torch.logsumexp(z, -1)
            w = torch.exp(z - lse[t][:, None]).view(kv, G, n)
            out[t], spread[t] = (w @ v[:, :n]).view(H, D), (w @ v[:, :n].abs()).view(H, D)
            slack[t] = size.max(-1).values * (D + 24) * 2.0 ** -24 + (n + 64) * 2.0 ** -24
    return out, lse, spread, slack


def key_weights(q, lse, pages, table, cu, lens, kv: int, scale: float):
    """[(page, row, weights [kv], error bound [kv])] of every key that a sequence with new tokens holds up to its last token."""
    T, H, D = q.shape
    found = []
    for b, L in enumerate(lens.tolist()):
        c0, c1 = int(cu[b]), min(int(cu[b + 1]), T)
        if c1 <= c0:
            continue
        base = L - int(cu[b + 1])
        p, k, _ = keys_of(pages, table, b, base + c1, kv, D)
        x = q[c0:c1].double().view(-1, kv, H // kv, D).permute(1, 0, 2, 3)
        z = torch.einsum("htgd,hjd->htgj", x, k) * scale
        size = torch.einsum("htgd,hjd->htgj", x.abs(), k.abs()) * scale
        ref = lse[c0:c1].double().view(-1, kv, H // kv).permute(1, 0, 2)[..., None]
        sees = p <= base + torch.arange(c0, c1, device=q.device)[:, None]
        e = torch.where(sees[:, None], torch.exp(z - ref), 0.0)
        off = torch.where(e > 0, e * (size * (D + 24) + ref.abs() * 4 + 8), 0.0) * 2.0 ** -24
        w = e.sum((1, 2))
        off = off.sum((1, 2)) + w * (e.shape[1] * e.shape[2] + 8) * 2.0 ** -24
        found += [(int(table[b, j // KEYS]), int(j % KEYS), w[:, i], off[:, i]) for i, j in enumerate(p.tolist())]
    return found


def kept(weights, table, b: int, n: int, keep: int, recent: int, room: int, n_pages: int, head: int):
    """The positions that stay, ascending."""
    at = {j: int(table[b, j // KEYS]) for j in range(max(0, min(n, table.shape[1] * KEYS)))}
    at = {j: page for j, page in at.items() if 0 <= page < n_pages}
    k = min(max(keep, 0), len(at), room)
    last = min(n, table.shape[1] * KEYS) - min(recent, k)
    sure = [j for j in at if j >= last]
    rest = [j for j in at if j < last]
    w = {j: float(weights[at[j], head, j % KEYS]) for j in rest}
    rest.sort(key=lambda j: (-math.inf if math.isnan(w[j]) else -w[j] if not math.isinf(w[j]) else (-1e300 if w[j] > 0 else 1e300), j))
    return sorted(sure + rest[:k - len(sure)])
