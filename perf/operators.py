"""Timed cases of the paged latent cache: attention of new tokens over it, writing it, reading it back, and the
residual norm that starts the block which fills it.

A KV page is 41216 bytes: 64 keys of 512 e4m3fn codes, their 64 fp32 scales, their 64 rope parts of 64 bf16.  The key
at position p of sequence b is row p % 64 of page ``block_table[b, p // 64]``; its latent is code * scale.  A batch is
``cu_seqlens`` (its sequences' token ranges) and ``seq_lens`` (the cache lengths with the new tokens), so the last new
token of a sequence stands at position seq_len - 1.

``run`` computes the operators in elementary torch operations in 32 bits, or, with ``own`` set, calls the
framework's.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BF16, F32, F64, FP8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
LATENT, ROPE, KEYS = 512, 64, 64
SCALE_AT, ROPE_AT = KEYS * LATENT, KEYS * LATENT + KEYS * 4
PAGE_BYTES = ROPE_AT + KEYS * ROPE * 2
EPS = 1e-6
SOFTMAX_SCALE = 192 ** -0.5 * (0.1 * math.log(40.0) + 1.0) ** 2  # DeepSeek-V3.2: 128 + 64 wide heads, rope factor 40


def listed() -> list[dict]:
    return [
        # one token of one short sequence: the smallest decode call, all latency
        {"name": "step_1", "kind": "attn", "heads": 16, "seqs": 1, "new": 1, "total": 500, "ragged": False, "lens": 0, "pad": 0},
        # one sequence at a 128K context, a token with its three drafts
        {"name": "step_128k", "kind": "attn", "heads": 16, "seqs": 1, "new": 4, "total": 131072, "ragged": False, "lens": 0, "pad": 0},
        # a decode batch with contexts of all lengths, padded to the size that its graph was captured for
        {"name": "batch_60", "kind": "attn", "heads": 16, "seqs": 60, "new": 1, "total": 32768, "ragged": True, "lens": 1, "pad": 4},
        # all 128 heads on one GPU, a small batch
        {"name": "heads_128", "kind": "attn", "heads": 128, "seqs": 8, "new": 1, "total": 16384, "ragged": True, "lens": 2, "pad": 0},
        # a prefill chunk over an earlier context
        {"name": "chunk_2048", "kind": "attn", "heads": 16, "seqs": 1, "new": 2048, "total": 16384, "ragged": False, "lens": 0, "pad": 0},
        # prompts and decodes in one batch, odd lengths, the head count of a seven-way split
        {"name": "mixed_7", "kind": "attn", "heads": 20, "seqs": 7, "new": 700, "total": 5000, "ragged": True, "lens": 3, "pad": 0},
        # a decode step's new key
        {"name": "write_1", "kind": "write", "seqs": 1, "new": 1, "total": 1000, "ragged": False, "lens": 0, "pad": 0},
        # the keys of a large prefill step of several prompts
        {"name": "write_8000", "kind": "write", "seqs": 5, "new": 4000, "total": 9000, "ragged": True, "lens": 4, "pad": 13},
        # a sequence's cache handed to the sparse attention's flat form
        {"name": "read_2100", "kind": "read", "seqs": 1, "new": 2100, "total": 2100, "ragged": False, "lens": 0, "pad": 0},
        # the caches of a batch of long sequences
        {"name": "read_batch", "kind": "read", "seqs": 9, "new": 65536, "total": 65536, "ragged": True, "lens": 5, "pad": 0},
        # the hidden state of one token with its drafts between two layers
        {"name": "norm_4", "kind": "norm", "rows": 4, "dim": 7168},
        # a prefill chunk's hidden states
        {"name": "norm_4096", "kind": "norm", "rows": 4096, "dim": 7168},
    ]


MAX_SCORES = 16384 * 16 * 2048  # rows times keys of the largest listed attention, padded
MAX_KEYS = 300_000              # cached keys of a drawn case


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("attn", "attn", "attn", "write", "read", "norm"))
    if kind == "norm":
        return {"kind": kind, "rows": _log_int(rng, 1, 4096), "dim": rng.choice((7168, 6144, 2048, 1536))}
    seqs = _log_int(rng, 1, 64)
    case = {"kind": kind, "seqs": seqs, "ragged": seqs > 1 and rng.random() < 0.8, "lens": rng.randrange(1 << 30),
            "pad": rng.choice((0, 0, 0, 1, 7))}
    if kind == "attn":
        heads = rng.choice((8, 10, 16, 16, 20, 128))
        new = rng.choice((1, 1, 2, 4, _log_int(rng, 5, 2048), _log_int(rng, 5, 2048)))
        total = max(new, min(_log_int(rng, 32, 131072), MAX_KEYS // seqs, MAX_SCORES // (seqs * new * heads)))
        new = max(1, min(new, MAX_SCORES // (seqs * total * heads)))
        return {**case, "heads": heads, "new": new, "total": total}
    if kind == "write":
        new = min(_log_int(rng, 1, 4096), max(1, 8192 // seqs))
        return {**case, "new": new, "total": new + _log_int(rng, 1, 8192)}
    total = min(_log_int(rng, 32, 65536), MAX_KEYS // seqs)
    return {**case, "new": total, "total": total}


def _lengths(case) -> tuple[list[int], list[int]]:
    """New tokens and cache length of every sequence; the first has the largest of both."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["new"]] * n, [case["total"]] * n
    r = random.Random(case["lens"])
    new = [case["new"]] + [_log_int(r, 1, case["new"]) for _ in range(n - 1)]
    if case["kind"] == "read":
        return new, list(new)
    total = [case["total"]] + [_log_int(r, max(1, case["total"] // 16), case["total"]) for _ in range(n - 1)]
    return new, [max(a, b) for a, b in zip(new, total)]


def _paged(case, g):
    """A batch's metadata over pages in random order, two pages to spare."""
    new, total = _lengths(case)
    pages = [-(-t // KEYS) for t in total]
    order = torch.randperm(sum(pages) + 2, generator=g, device=DEV).to(torch.int32)
    used = torch.arange(max(pages), device=DEV) < torch.tensor(pages, device=DEV)[:, None]
    table = torch.zeros(len(new), max(pages), dtype=torch.int32, device=DEV)
    table[used] = order[:sum(pages)]
    cu = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    return {"table": table, "cu": cu, "lens": torch.tensor(total, dtype=torch.int32, device=DEV), "n_pages": order.numel(),
            "tokens": sum(new) + case["pad"], "max_new": max(new), "max_len": max(total), "case": case}


def _views(pages):
    """The codes, scales and rope parts of pages, as views."""
    n = pages.shape[0]
    return (pages[:, :SCALE_AT].view(n, KEYS, LATENT), pages[:, SCALE_AT:ROPE_AT].view(F32),
            pages[:, ROPE_AT:].view(BF16).view(n, KEYS, ROPE))


def _filled(n_pages: int, g):
    """Pages of normalised latents, N(0, 1), as a running server's pool holds them: quantised per key."""
    pages = torch.empty(n_pages, PAGE_BYTES, dtype=torch.uint8, device=DEV)
    codes, scales, rope = _views(pages)
    v = torch.randn(n_pages, KEYS, LATENT, generator=g, device=DEV)
    scales.copy_(v.abs().amax(-1) / 448)
    codes.copy_(v.div_(scales[..., None]).clamp_(-448, 448).to(FP8).view(torch.uint8))
    rope.copy_(torch.randn(n_pages, KEYS, ROPE, generator=g, device=DEV))
    return pages


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    if case["kind"] == "norm":
        rows, dim = case["rows"], case["dim"]
        return {"case": case, "x": normal(rows, dim), "residual": normal(rows, dim, std=3.0),
                "gamma": torch.rand(dim, generator=g, device=DEV) * 0.2 + 0.9,
                "sum": torch.zeros(rows, dim, dtype=BF16, device=DEV), "y": torch.zeros(rows, dim, dtype=BF16, device=DEV),
                "q": torch.zeros(rows, dim, dtype=FP8, device=DEV), "s": torch.zeros(rows, dim // 128, device=DEV),
                "logs": torch.zeros(1, dtype=torch.uint8, device=DEV)}
    st = _paged(case, g)
    st["pages"] = _filled(st["n_pages"], g)
    T = st["tokens"]
    if case["kind"] == "attn":
        H = case["heads"]
        return {**st, "q": normal(T, H, LATENT, std=0.5), "q_pe": normal(T, H, ROPE, std=0.5),
                "out": torch.zeros(T, H, LATENT, dtype=BF16, device=DEV), "lse": torch.zeros(T, H, device=DEV)}
    if case["kind"] == "write":
        angle = torch.rand(T, 1, ROPE // 2, generator=g, device=DEV, dtype=F64) * (2 * math.pi)
        return {**st, "kv": normal(T, LATENT), "pe": normal(T, ROPE),
                "gamma": torch.rand(LATENT, generator=g, device=DEV) * 0.2 + 0.9,
                "freqs": torch.stack([angle.cos(), angle.sin()], -1).to(F32).reshape(T, 1, ROPE)}
    return {**st, "kv": torch.zeros(T, LATENT, dtype=BF16, device=DEV), "pe": torch.zeros(T, ROPE, dtype=BF16, device=DEV)}


# ------------------------------------------------------------------------------------------- the operators
def _slots(st):
    """The padded batch: token indices [B, max_new], which of them are there, and their positions."""
    i = torch.arange(st["max_new"], device=DEV)
    n = st["cu"][1:] - st["cu"][:-1]
    there = i < n[:, None]
    return (st["cu"][:-1, None] + i).long(), there, (st["lens"] - n)[:, None] + i


def _attention(st):
    B, H = st["table"].shape[0], st["case"]["heads"]
    token, there, pos = _slots(st)
    token = torch.where(there, token, 0)
    codes, scales, rope = _views(st["pages"])
    j = torch.arange(st["max_len"], device=DEV)
    page, row = st["table"].long()[:, j // KEYS], j % KEYS
    key = torch.cat([codes.view(FP8)[page, row].to(F32) * scales[page, row][..., None], rope[page, row].to(F32)], -1)
    key = torch.where((j < st["lens"][:, None])[..., None], key, 0.0)
    q = torch.cat([st["q"], st["q_pe"]], -1)[token].to(F32).reshape(B, -1, LATENT + ROPE)
    score = torch.bmm(q, key.transpose(1, 2).contiguous()).mul_(SOFTMAX_SCALE).view(B, st["max_new"], H, -1)
    score.masked_fill_((j > pos[..., None])[:, :, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    out = torch.bmm(p.view(B, -1, p.shape[-1]), key[..., :LATENT].contiguous()).view(B, st["max_new"], H, LATENT)
    out = torch.where(total > 0, out / total, 0.0)
    st["out"][token[there]] = out[there].to(BF16)
    st["lse"][token[there]] = (top + total.log()).squeeze(-1)[there]
    return st["out"], st["lse"]


def _write(st):
    token, there, pos = _slots(st)
    t, pos = token[there], pos[there].long()
    b = torch.arange(st["table"].shape[0], device=DEV)[:, None].expand_as(there)[there]
    page, row = st["table"].long()[b, pos // KEYS], pos % KEYS
    codes, scales, rope = _views(st["pages"])
    x = st["kv"][t].to(F32)
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * st["gamma"]
    s = n.abs().amax(-1).clamp_min(1e-4) / 448
    codes[page, row] = (n / s[:, None]).clamp(-448, 448).to(FP8).view(torch.uint8)
    scales[page, row] = s
    z, w = st["pe"][t].to(F32).view(-1, ROPE // 2, 2), st["freqs"][t].view(-1, ROPE // 2, 2)
    rope[page, row] = torch.stack([z[..., 0] * w[..., 0] - z[..., 1] * w[..., 1],
                                   z[..., 0] * w[..., 1] + z[..., 1] * w[..., 0]], -1).to(BF16).view(-1, ROPE)


def _read(st):
    token, there, pos = _slots(st)
    t, pos = token[there], pos[there].long()
    b = torch.arange(st["table"].shape[0], device=DEV)[:, None].expand_as(there)[there]
    page, row = st["table"].long()[b, pos // KEYS], pos % KEYS
    codes, scales, rope = _views(st["pages"])
    st["kv"][t] = (codes.view(FP8)[page, row].to(F32) * scales[page, row][:, None]).to(BF16)
    st["pe"][t] = rope[page, row]


def _norm(st):
    h = st["x"].to(F32) + st["residual"].to(F32)
    n = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * st["gamma"]
    group = n.view(*n.shape[:-1], -1, 128)
    s = group.abs().amax(-1).clamp_min(1e-4) / 448
    return h.to(BF16), n.to(BF16), (group / s[..., None]).clamp(-448, 448).to(FP8).view(n.shape), s


def run(st):
    kind = st["case"]["kind"]
    if own:
        if kind == "norm":
            from tilert_amd.rmsnorm import add_rmsnorm_quant
            add_rmsnorm_quant(st["x"], st["residual"], st["gamma"], st["sum"], st["y"], st["q"], st["s"], st["logs"],
                              model_arch="deepseek_v3_2", scale_fmt="div")
            return st["sum"], st["y"], st["q"], st["s"]
        batch = (st["pages"], st["table"], st["cu"], st["lens"])
        if kind == "attn":
            from tilert_amd.flash_paged_mla import flash_paged_mla
            flash_paged_mla(st["q"], st["q_pe"], *batch, st["out"], st["lse"], model_arch="deepseek_v3_2")
            return st["out"], st["lse"]
        from tilert_amd.mla_cache import mla_cache_read, mla_cache_write
        if kind == "write":
            mla_cache_write(st["kv"], st["pe"], *batch, st["gamma"], st["freqs"], scale_fmt="div")
        else:
            mla_cache_read(*batch, st["kv"], st["pe"])
    elif kind == "norm":
        return _norm(st)
    elif kind == "attn":
        return _attention(st)
    else:
        (_write if kind == "write" else _read)(st)
    if kind == "read":
        return st["kv"], st["pe"]
    codes, scales, rope = _views(st["pages"])
    return codes.view(FP8), scales, rope


# --------------------------------------------------------------------------------------- work, and 64 bits
def work(case):
    if case["kind"] == "norm":
        n = case["rows"] * case["dim"]
        return {"bytes": n * (2 + 2 + 2 + 2 + 1 + 4 / 128) + case["dim"] * 4, "flops": n * 8}
    new, total = _lengths(case)
    T = sum(new)
    if case["kind"] == "write":
        return {"bytes": T * (2 * (LATENT + ROPE) + 4 * ROPE + LATENT + 4 + 2 * ROPE) + 4 * LATENT, "flops": T * LATENT * 6}
    if case["kind"] == "read":
        return {"bytes": T * (LATENT + 4 + 2 * ROPE + 2 * (LATENT + ROPE)), "flops": T * LATENT}
    H = case["heads"]
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, total))
    return {"bytes": sum(total) * (LATENT + 4 + 2 * ROPE) + T * H * (2 * (LATENT + ROPE) + 2 * LATENT + 4),
            "flops": 2 * H * seen * (2 * LATENT + ROPE)}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        h = st["x"].double() + st["residual"].double()
        n = h / torch.sqrt((h * h).mean(1, keepdim=True) + EPS) * st["gamma"].double()
        s = n.view(case["rows"], -1, 128).abs().amax(2).clamp(min=1e-4) / 448.0
        return h, n, n / s.repeat_interleave(128, 1), s
    codes, scales, rope = _views(st["pages"])
    cu, lens, table = st["cu"].tolist(), st["lens"].tolist(), st["table"].long()

    def keys(b, first, last):
        p = torch.arange(first, last, device=DEV)
        return table[b][torch.div(p, KEYS, rounding_mode="floor")], p.remainder(KEYS)

    if case["kind"] == "attn":
        out, lse = st["out"].double(), st["lse"].double()
        for b, L in enumerate(lens):
            at = keys(b, 0, L)
            latent = codes.view(FP8)[at].double() * scales[at].double().unsqueeze(1)
            pe = rope[at].double()
            base = L - (cu[b + 1] - cu[b])
            step = max(1, (1 << 27) // (L * case["heads"]))
            for t0 in range(cu[b], cu[b + 1], step):
                t1 = min(t0 + step, cu[b + 1])
                z = st["q"][t0:t1].double() @ latent.T + st["q_pe"][t0:t1].double() @ pe.T
                p = torch.arange(base + t0 - cu[b], base + t1 - cu[b], device=DEV)
                hidden = torch.arange(L, device=DEV) > p.view(-1, 1, 1)
                z = (z * SOFTMAX_SCALE).masked_fill(hidden, -math.inf)
                lse[t0:t1] = torch.logsumexp(z, -1)
                out[t0:t1] = torch.exp(z - lse[t0:t1].unsqueeze(-1)) @ latent
        return out, lse
    if case["kind"] == "read":
        kv, pe = st["kv"].double(), st["pe"].double()
        for b, L in enumerate(lens):
            at = keys(b, L - (cu[b + 1] - cu[b]), L)
            kv[cu[b]:cu[b + 1]] = codes.view(FP8)[at].double() * scales[at].double().unsqueeze(1)
            pe[cu[b]:cu[b + 1]] = rope[at].double()
        return kv, pe
    quotient, scale, turned = codes.view(FP8).double(), scales.double(), rope.double()
    x = st["kv"].double()
    n = x / torch.sqrt((x * x).mean(1, keepdim=True) + EPS) * st["gamma"].double()
    s = n.abs().amax(1).clamp(min=1e-4) / 448.0
    z = torch.view_as_complex(st["pe"].double().view(-1, ROPE // 2, 2))
    z = torch.view_as_real(z * torch.view_as_complex(st["freqs"].double().view(-1, ROPE // 2, 2))).view(-1, ROPE)
    for b, L in enumerate(lens):
        t, at = slice(cu[b], cu[b + 1]), keys(b, L - (cu[b + 1] - cu[b]), L)
        quotient[at], scale[at], turned[at] = n[t] / s[t].unsqueeze(1), s[t], z[t]
    return quotient, scale, turned
