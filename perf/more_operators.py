"""Timed cases of the paged per-head cache (grouped-query attention): norm, rotation and writing of new tokens, attention
over the cache, accumulated attention weights of its keys, and eviction by them.

A page holds 64 keys.  For each of its kv heads: 64 x D e4m3fn key codes, then D x 64 e4m3fn value codes (a value's dim is
its row); behind all heads two fp32 scales a head (keys, values), powers of two, padded to 128 bytes.  The key at position p
of sequence b is row p % 64 of page ``table[b, p // 64]``.  A batch is ``cu`` (its sequences' token ranges) and ``lens``
(the cache lengths with the new tokens), so the last new token of a sequence stands at position len - 1.

``run`` computes the operators in elementary torch operations in 32 bits, or, with ``own`` set, calls the
framework's.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
BF16, F32, F64, I32, FP8, U8 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.float8_e4m3fn, torch.uint8
KEYS = 64
EPS = 1e-6


def listed() -> list[dict]:
    one = {"ragged": False, "lens": 0, "pad": 0}
    return [
        # one token of one short sequence: the smallest decode call, all latency
        {"name": "step_1", "kind": "attn", "heads": 32, "kv": 8, "dim": 128, "seqs": 1, "new": 1, "total": 500, **one},
        # one sequence at a 128K context, a token with its three drafts
        {"name": "step_128k", "kind": "attn", "heads": 64, "kv": 8, "dim": 128, "seqs": 1, "new": 4, "total": 131072, **one},
        # a decode batch with contexts of all lengths, padded to the size that its graph was captured for
        {"name": "batch_60", "kind": "attn", "heads": 64, "kv": 8, "dim": 128, "seqs": 60, "new": 1, "total": 32768, "ragged": True,
         "lens": 1, "pad": 4},
        # a prefill chunk over an earlier context
        {"name": "chunk_2048", "kind": "attn", "heads": 32, "kv": 8, "dim": 128, "seqs": 1, "new": 2048, "total": 16384, **one},
        # prompts and decodes in one batch: odd lengths, five query heads to a kv head, narrow heads
        {"name": "mixed_7", "kind": "attn", "heads": 20, "kv": 4, "dim": 64, "seqs": 7, "new": 700, "total": 5000, "ragged": True,
         "lens": 3, "pad": 0},
        # a decode step's new token
        {"name": "write_1", "kind": "write", "heads": 32, "kv": 8, "dim": 128, "rope": 128, "seqs": 1, "new": 1, "total": 1000, **one},
        # the tokens of a large prefill step of several prompts, half of a head's dims rotated
        {"name": "write_8000", "kind": "write", "heads": 32, "kv": 8, "dim": 128, "rope": 64, "seqs": 5, "new": 4000, "total": 9000,
         "ragged": True, "lens": 4, "pad": 13},
        # a decode batch's weights, each step
        {"name": "sums_60", "kind": "sums", "heads": 64, "kv": 8, "dim": 128, "seqs": 60, "new": 1, "total": 32768, "ragged": True,
         "lens": 1, "pad": 4},
        # the weights of a prefill chunk's queries
        {"name": "sums_2048", "kind": "sums", "heads": 32, "kv": 8, "dim": 128, "seqs": 1, "new": 2048, "total": 16384, **one},
        # a prompt's last queries, few rows over few pages
        {"name": "sums_32", "kind": "sums", "heads": 20, "kv": 4, "dim": 64, "seqs": 2, "new": 32, "total": 1500, **one},
        # a short sequence brought down to half
        {"name": "evict_4000", "kind": "evict", "kv": 4, "dim": 128, "seqs": 1, "total": 4000, "keep": 2000, "recent": 32, "ragged": False,
         "lens": 0},
        # a batch of long sequences of all lengths, each brought down to the same size
        {"name": "evict_batch", "kind": "evict", "kv": 8, "dim": 128, "seqs": 9, "total": 65536, "keep": 8192, "recent": 256, "ragged": True,
         "lens": 5},
    ]


LAYOUTS = ((32, 8), (64, 8), (16, 2), (20, 4), (8, 8), (28, 4), (128, 1), (24, 1))  # query heads, kv heads
MAX_SCORES = 16384 * 32 * 2048   # rows times keys of the largest listed attention, padded
MAX_VALUES = 300_000 * 8 * 128   # cached values of a drawn case: keys times kv heads times dims, keys alone


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(("attn", "attn", "attn", "write", "sums", "sums", "evict"))
    heads, kv = rng.choice(LAYOUTS)
    dim = rng.choice((64, 128, 128))
    seqs = _log_int(rng, 1, 64)
    case = {"kind": kind, "kv": kv, "dim": dim, "seqs": seqs, "ragged": seqs > 1 and rng.random() < 0.8, "lens": rng.randrange(1 << 30)}
    room = MAX_VALUES // (seqs * kv * dim)
    if kind == "evict":
        total = max(2, min(_log_int(rng, 100, 65536), room))
        keep = _log_int(rng, 1, total)
        return {**case, "total": total, "keep": keep, "recent": rng.choice((0, keep // 2, min(keep, 64)))}
    case.update(heads=heads, pad=rng.choice((0, 0, 0, 1, 7)))
    if kind == "write":
        new = min(_log_int(rng, 1, 4096), max(1, 8192 // seqs))
        return {**case, "rope": rng.choice((dim, dim, dim // 2)), "new": new, "total": new + _log_int(rng, 1, 4096)}
    new = rng.choice((1, 1, 2, 4, _log_int(rng, 5, 2048), _log_int(rng, 5, 2048)))
    total = max(new, min(_log_int(rng, 32, 131072), room, MAX_SCORES // (seqs * new * heads)))
    new = max(1, min(new, MAX_SCORES // (seqs * total * heads)))
    return {**case, "new": new, "total": total}


def _lengths(case) -> tuple[list[int], list[int]]:
    """New tokens and cache length of every sequence; the first has the largest of both."""
    n, most = case["seqs"], case.get("new", 0)
    if not case["ragged"]:
        return [most] * n, [case["total"]] * n
    r = random.Random(case["lens"])
    new = [most] + [_log_int(r, 1, most) if most else 0 for _ in range(n - 1)]
    total = [case["total"]] + [_log_int(r, max(1, case["total"] // 16), case["total"]) for _ in range(n - 1)]
    return new, [max(a, b) for a, b in zip(new, total)]


def page_bytes(kv: int, dim: int) -> int:
    return kv * 2 * KEYS * dim + -(-kv * 8 // 128) * 128


def _views(pages, kv: int, dim: int):
    """The key codes [n, kv, 64, dim], value codes [n, kv, dim, 64] and scales [n, kv, 2] of pages, as views."""
    n, codes = pages.shape[0], kv * 2 * KEYS * dim
    both = pages[:, :codes].view(n, kv, 2, KEYS * dim)
    return (both[:, :, 0].view(n, kv, KEYS, dim), both[:, :, 1].view(n, kv, dim, KEYS),
            pages[:, codes:codes + kv * 8].view(F32).view(n, kv, 2))


def _scale_for(amax):
    """The least power of two s with max(amax, 1e-4) <= 448 s."""
    mantissa, exponent = torch.frexp(amax.clamp_min(1e-4))  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    return torch.ldexp(torch.ones_like(mantissa), exponent - 9 + (mantissa > 0.875))


def _codes(v, scale):
    return (v / scale).clamp(-448, 448).to(FP8).view(U8)


def _table(pages, order, first):
    """Tables of sequences with `pages` pages each, from `order` on from `first`."""
    used = torch.arange(max(max(pages), 1), device=DEV) < torch.tensor(pages, device=DEV)[:, None]
    table = torch.zeros(used.shape, dtype=I32, device=DEV)
    table[used] = order[first:first + sum(pages)]
    return table


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kv, dim, kind = case["kv"], case["dim"], case["kind"]
    new, total = _lengths(case)

    def normal(*shape, std=1.0, dtype=BF16):
        return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)

    # pages in random order, two to spare, filled as a running server's pool is: normalised keys, values of the same size
    here = [-(-t // KEYS) for t in total]
    kept = [-(-min(t, case["keep"]) // KEYS) for t in total] if kind == "evict" else [0]
    n = sum(here) + sum(kept) + 2
    order = torch.randperm(n, generator=g, device=DEV).to(I32)
    pages = torch.zeros(n, page_bytes(kv, dim), dtype=U8, device=DEV)
    k, v, scales = _views(pages, kv, dim)
    for i, codes in enumerate((k, v)):
        x = torch.randn(codes.shape, generator=g, device=DEV)
        scales[..., i] = _scale_for(x.abs().amax((-2, -1)))
        codes.copy_(_codes(x, scales[:, :, i, None, None]))
        del x
    st = {"case": case, "pages": pages, "table": _table(here, order, 0), "lens": torch.tensor(total, dtype=I32, device=DEV), "max_len": max(total)}
    if kind == "evict":
        return {**st, "weights": (torch.randn(n, kv, KEYS, generator=g, device=DEV) * 2).exp_(),
                "keep": torch.full((len(total),), case["keep"], dtype=I32, device=DEV), "kept_table": _table(kept, order, sum(here)),
                "kept": torch.zeros(len(total), dtype=I32, device=DEV), "slots": torch.zeros(len(total), kv, max(kept) * KEYS, dtype=I32, device=DEV)}
    heads, T = case["heads"], sum(new) + case["pad"]
    st.update(cu=torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=I32, device=DEV), max_new=max(new))
    if kind == "write":
        # the projections' joint output, whose heads the views name
        qkv = normal(T, (heads + 2 * kv) * dim)
        q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([heads * dim, kv * dim, kv * dim], 1))
        angle = torch.rand(T, 1, case["rope"] // 2, generator=g, device=DEV, dtype=F64) * (2 * math.pi)
        return {**st, "q": q, "k": k, "v": v, "freqs": torch.stack([angle.cos(), angle.sin()], -1).to(F32).reshape(T, 1, -1),
                "gamma_q": torch.rand(dim, generator=g, device=DEV) * 0.2 + 0.9, "gamma_k": torch.rand(dim, generator=g, device=DEV) * 0.2 + 0.9,
                "out": torch.zeros(T, heads, dim, dtype=BF16, device=DEV)}
    st.update(q=normal(T, heads, dim), lse=torch.zeros(T, heads, device=DEV))
    if kind == "attn":
        return {**st, "out": torch.zeros(T, heads, dim, dtype=BF16, device=DEV)}
    token, there, _ = _slots(st)
    st["lse"][token[there]] = torch.logsumexp(_scores(st), -1).view(len(new), kv, max(new), -1).transpose(1, 2).flatten(2)[there]
    return {**st, "weights": torch.zeros(n, kv, KEYS, device=DEV)}


# ------------------------------------------------------------------------------------------- the operators
def _slots(st):
    """The padded batch: token indices [B, max_new], which of them are there, and their positions."""
    i = torch.arange(st["max_new"], device=DEV)
    n = st["cu"][1:] - st["cu"][:-1]
    there = i < n[:, None]
    return torch.where(there, st["cu"][:-1, None] + i, 0).long(), there, (st["lens"] - n)[:, None] + i


def _places(st):
    """The padded caches: the page and row of positions [B, max_len], and which of them hold a key."""
    j = torch.arange(st["max_len"], device=DEV)
    return st["table"].long()[:, j // KEYS], (j % KEYS).expand(st["table"].shape[0], -1), j < st["lens"][:, None]


def _gather(codes, scales, page, row, there):
    """Cached keys or values [B, kv, max_len, dim] in fp32."""
    x = codes[page, :, row].view(FP8).to(F32) * scales[page][..., None]  # [B, max_len, kv, dim]
    return torch.where(there[..., None, None], x, 0.0).transpose(1, 2).contiguous()


def _scores(st):
    """Scores [B, kv, max_new * group, max_len], -inf where a row does not see a key."""
    case = st["case"]
    token, there, pos = _slots(st)
    page, row, valid = _places(st)
    k, _, scales = _views(st["pages"], case["kv"], case["dim"])
    key = _gather(k, scales[..., 0], page, row, valid)
    B, N = token.shape
    q = st["q"][token].to(F32).view(B, N, case["kv"], -1, case["dim"]).transpose(1, 2).reshape(B * case["kv"], -1, case["dim"])
    s = torch.bmm(q, key.flatten(0, 1).transpose(1, 2).contiguous()).mul_(case["dim"] ** -0.5).view(B, case["kv"], N, -1, key.shape[2])
    hidden = torch.arange(st["max_len"], device=DEV) > torch.where(there, pos, -1)[..., None]
    return s.masked_fill_(hidden[:, None, :, None], -math.inf).flatten(2, 3)


def _attention(st):
    case = st["case"]
    token, there, _ = _slots(st)
    s = _scores(st)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    del s
    total = p.sum(-1, keepdim=True)
    _, v, scales = _views(st["pages"], case["kv"], case["dim"])
    value = _gather(v.transpose(2, 3), scales[..., 1], *_places(st))
    out = torch.bmm(p.flatten(0, 1), value.flatten(0, 1)).view(*p.shape[:3], -1)
    out = torch.where(total > 0, out / total, 0.0)
    B, N = token.shape
    out = out.view(B, case["kv"], N, -1, case["dim"]).transpose(1, 2).flatten(2, 3)
    lse = (top + total.log()).view(B, case["kv"], N, -1).transpose(1, 2).flatten(2)
    st["out"][token[there]] = out[there].to(BF16)
    st["lse"][token[there]] = lse[there]
    return st["out"], st["lse"]


def _sums(st):
    case = st["case"]
    token, _, _ = _slots(st)
    B, N = token.shape
    lse = st["lse"][token].view(B, N, case["kv"], -1).transpose(1, 2).reshape(B, case["kv"], -1, 1)
    w = torch.exp(_scores(st).sub_(lse)).sum(2)  # a row that is not there sees nothing
    page, row, valid = _places(st)
    st["weights"][page[valid], :, row[valid]] = w.transpose(1, 2)[valid]
    return st["weights"]


def _turned(x, gamma, freqs):
    x = x.to(F32)
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * gamma
    half = freqs.shape[-1] // 2
    c, s = freqs[..., 0::2], freqs[..., 1::2]
    a, b = n[..., :half], n[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, n[..., 2 * half:]], -1)


def _write(st):
    case = st["case"]
    kv, dim = case["kv"], case["dim"]
    token, there, pos = _slots(st)
    t, p = token[there], pos[there].long()
    b = torch.arange(st["table"].shape[0], device=DEV)[:, None].expand_as(there)[there]
    page, row = st["table"].long()[b, p // KEYS], p % KEYS
    st["out"][t] = _turned(st["q"][t], st["gamma_q"], st["freqs"][t]).to(BF16)
    y = torch.stack([_turned(st["k"][t], st["gamma_k"], st["freqs"][t]), st["v"][t].to(F32)])  # [2, tokens, kv, dim]
    k, v, scales = _views(st["pages"], kv, dim)
    # a block's scale: what its new rows need, and no less than that of the older keys in front of them
    amax = torch.zeros(2, k.shape[0], kv, device=DEV).scatter_reduce_(1, page[None, :, None].expand(2, -1, kv), y.abs().amax(-1), "amax")
    need, touched = _scale_for(amax), torch.zeros(k.shape[0], dtype=torch.bool, device=DEV)
    touched[page] = True
    older = torch.zeros(k.shape[0], dtype=torch.long, device=DEV)  # older keys of a touched page
    first = (st["lens"] - (st["cu"][1:] - st["cu"][:-1])).long()
    began = st["table"].long().gather(1, (first // KEYS)[:, None])[:, 0]
    older[began] = first % KEYS
    old = scales.permute(2, 0, 1)
    s = torch.where((older > 0)[None, :, None], torch.maximum(old, need), need)
    at = older.nonzero()[:, 0]
    is_old = torch.arange(KEYS, device=DEV) < older[at, None]
    back = (old / s)[:, at, :, None, None]
    k[at] = torch.where(is_old[:, None, :, None], (k[at].view(FP8).to(F32) * back[0]).to(FP8).view(U8), k[at])
    v[at] = torch.where(is_old[:, None, None, :], (v[at].view(FP8).to(F32) * back[1]).to(FP8).view(U8), v[at])
    code = _codes(y, s[:, page][..., None])
    k[page, :, row] = code[0]
    v[page, :, :, row] = code[1]
    scales[touched] = s[:, touched].permute(1, 2, 0)


def _evict(st):
    case = st["case"]
    kv, dim, recent = case["kv"], case["dim"], case["recent"]
    page, row, valid = _places(st)
    n, keep = st["lens"][:, None, None], torch.minimum(st["lens"], st["keep"])
    j = torch.arange(st["max_len"], device=DEV)
    last = j >= n - torch.minimum(keep, torch.full_like(keep, recent))[:, None, None]
    w = st["weights"][page, :, row].transpose(1, 2)                                       # [B, kv, max_len]
    rank = torch.where(valid[:, None], torch.where(last, math.inf, w), -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :st["slots"].shape[2]]  # ties: the lowest first
    held = torch.arange(order.shape[2], device=DEV) < keep[:, None, None]
    slots = torch.where(held, order, 1 << 30).sort(-1).values
    slots = torch.nn.functional.pad(slots, (0, st["slots"].shape[2] - slots.shape[2]), value=1 << 30)
    held = slots < 1 << 30
    st["slots"].copy_(torch.where(held, slots, -1))
    st["kept"].copy_(keep)
    B, _, K = slots.shape
    src = torch.where(held, slots, 0)
    from_page = page.gather(1, src.flatten(1)).view(src.shape)
    from_row, h = src % KEYS, torch.arange(kv, device=DEV)[:, None]
    k, v, scales = _views(st["pages"], kv, dim)
    s = scales[from_page, h]                                                               # [B, kv, K, 2]
    x = torch.stack([k[from_page, h, from_row], v.transpose(2, 3)[from_page, h, from_row]]).view(FP8).to(F32) * s.permute(3, 0, 1, 2)[..., None]
    x = torch.where(held[..., None], x, 0.0).view(2, B, kv, K // KEYS, KEYS, dim)
    new_s = _scale_for(x.abs().amax((-2, -1)))                                             # [2, B, kv, K / 64]
    code = _codes(x, new_s[..., None, None])
    wt = st["weights"][from_page, h, from_row].view(B, kv, -1, KEYS)
    held = held.view(B, kv, -1, KEYS)
    to = st["kept_table"].long()
    used = held[:, 0].any(-1)
    into, mine = to[used], lambda a: a.transpose(1, 2)[used]                               # [blocks, kv, ..]
    there = mine(held)
    k[into] = torch.where(there[..., None], mine(code[0]), k[into])
    v[into] = torch.where(there[:, :, None], mine(code[1]).transpose(2, 3), v[into])
    scales[into] = torch.stack([mine(new_s[0]), mine(new_s[1])], -1)
    st["weights"][into] = torch.where(there, mine(wt), st["weights"][into])


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if own:
        from tilert_amd.flash_paged_gqa import flash_paged_gqa
        from tilert_amd.gqa_cache import gqa_cache_evict, gqa_cache_weights, gqa_cache_write
        if kind == "evict":
            gqa_cache_evict(st["pages"], st["weights"], st["table"], st["lens"], st["keep"], st["kept_table"], st["kept"], st["slots"],
                            head_dim=case["dim"], recent=case["recent"])
        else:
            batch = (st["pages"], st["table"], st["cu"], st["lens"])
            if kind == "attn":
                flash_paged_gqa(st["q"], *batch, st["out"], st["lse"], kv_heads=case["kv"])
            elif kind == "sums":
                gqa_cache_weights(st["q"], st["lse"], *batch, st["weights"], accumulate=False)
            else:
                gqa_cache_write(st["k"], st["v"], *batch, st["gamma_k"], st["freqs"], query=st["q"], gamma_q=st["gamma_q"],
                                query_out=st["out"], eps=EPS)
    else:
        {"attn": _attention, "sums": _sums, "write": _write, "evict": _evict}[kind](st)
    if kind == "attn":
        return st["out"], st["lse"]
    if kind == "sums":
        return st["weights"]
    k, v, scales = _views(st["pages"], case["kv"], case["dim"])
    if kind == "write":
        return st["out"], k.view(FP8), v.view(FP8), scales
    return st["kept"], st["slots"], k.view(FP8), v.view(FP8), scales, st["weights"]


# --------------------------------------------------------------------------------------- work, and 64 bits
def work(case):
    new, total = _lengths(case)
    kv, dim = case["kv"], case["dim"]
    if case["kind"] == "evict":
        kept = sum(min(t, case["keep"]) for t in total) * kv
        return {"bytes": sum(total) * kv * 4 + kept * (4 * dim + 8), "flops": kept * dim * 8}
    T, heads = sum(new), case["heads"]
    if case["kind"] == "write":
        return {"bytes": T * (heads * dim * 4 + kv * dim * 6 + case["rope"] * 4) + 8 * dim, "flops": T * dim * (heads + 2 * kv) * 8}
    seen = sum(n * (L - n) + n * (n + 1) // 2 for n, L in zip(new, total))
    if case["kind"] == "sums":
        return {"bytes": sum(total) * kv * (dim + 4) + T * heads * (2 * dim + 4), "flops": 2 * heads * seen * dim}
    return {"bytes": sum(total) * kv * 2 * dim + T * heads * (4 * dim + 4), "flops": 4 * heads * seen * dim}


def exact(case, seed):
    st = prepare(case, seed)
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    k, v, scales = _views(st["pages"], kv, dim)
    lens, table = st["lens"].tolist(), st["table"].long()

    def keys(b, first, last):
        p = torch.arange(first, last, device=DEV)
        return table[b][torch.div(p, KEYS, rounding_mode="floor")], p.remainder(KEYS)

    def power(a):  # the least power of two s with max(a, 1e-4) <= 448 s
        return torch.exp2(torch.ceil(torch.log2(a.clamp(min=1e-4) / 448)))

    if kind == "evict":
        kept, slots, weights = st["kept"].double(), torch.full(st["slots"].shape, -1.0, dtype=F64, device=DEV), st["weights"].double()
        kc, vc, sc = k.view(FP8).double(), v.view(FP8).double(), scales.double()
        for b, L in enumerate(lens):
            n = min(L, case["keep"])
            r = min(case["recent"], n)
            page, row = keys(b, 0, L)
            kept[b] = n
            for h in range(kv):
                w = st["weights"][page, h, row].double()
                rest = torch.argsort(w[:L - r], descending=True, stable=True)[:n - r]
                at = torch.cat([rest.sort().values, torch.arange(L - r, L, device=DEV)])
                slots[b, h, :n] = at.double()
                for c in range(0, n, KEYS):
                    src, to = at[c:c + KEYS], int(st["kept_table"][b, c // KEYS])
                    m = src.numel()
                    key = k[page[src], h, row[src]].view(FP8).double() * scales[page[src], h, 0].double()[:, None]
                    val = v[page[src], h, :, row[src]].view(FP8).double() * scales[page[src], h, 1].double()[:, None]
                    sc[to, h, 0], sc[to, h, 1] = power(key.abs().amax()), power(val.abs().amax())
                    kc[to, h, :m], vc[to, h, :, :m] = key / sc[to, h, 0], (val / sc[to, h, 1]).T
                    weights[to, h, :m] = w[src]
        return None, None, kc, vc, sc, weights
    cu = st["cu"].tolist()
    if kind == "write":
        out, kc, vc, sc = st["out"].double(), k.view(FP8).double(), v.view(FP8).double(), scales.double()
        R = case["rope"]
        w = torch.view_as_complex(st["freqs"].double().view(-1, R // 2, 2))[:, None]

        def turned(x, gamma):
            x = x.double()
            n = x / torch.sqrt((x * x).mean(2, keepdim=True) + EPS) * gamma.double()
            z = torch.complex(n[..., :R // 2], n[..., R // 2:R]) * w
            return torch.cat([z.real, z.imag, n[..., R:]], 2)

        q, key, val = turned(st["q"], st["gamma_q"]), turned(st["k"], st["gamma_k"]), st["v"].double()
        for b, L in enumerate(lens):
            out[cu[b]:cu[b + 1]] = q[cu[b]:cu[b + 1]]
            first = L - (cu[b + 1] - cu[b])
            for c in range(first // KEYS, -(-L // KEYS)):
                lo, hi, pg = max(first, c * KEYS), min(L, (c + 1) * KEYS), int(table[b, c])
                t, r0, r1 = cu[b] + lo - first, lo - c * KEYS, hi - c * KEYS
                for x, codes, i in ((key[t:t + hi - lo], kc[pg], 0), (val[t:t + hi - lo], vc[pg].transpose(1, 2), 1)):
                    x = x.transpose(0, 1)
                    s = power(x.abs().amax((1, 2)))
                    if r0:
                        s = torch.maximum(s, sc[pg, :, i])
                        codes[:, :r0] *= (sc[pg, :, i] / s)[:, None, None]
                    codes[:, r0:r1] = x / s[:, None, None]
                    sc[pg, :, i] = s
        return out, kc, vc, sc
    heads, group = case["heads"], case["heads"] // kv
    out, lse = st["q"].double() * 0, st["lse"].double()
    weights = torch.zeros(k.shape[0], kv, KEYS, dtype=F64, device=DEV)
    for b, L in enumerate(lens):
        page, row = keys(b, 0, L)
        base = L - (cu[b + 1] - cu[b])
        step = max(1, (1 << 27) // (L * group))
        for h in range(kv):
            key = k[page, h, row].view(FP8).double() * scales[page, h, 0].double()[:, None]
            val = v[page, h, :, row].view(FP8).double() * scales[page, h, 1].double()[:, None]
            mine = slice(h * group, (h + 1) * group)
            for t0 in range(cu[b], cu[b + 1], step):
                t1 = min(t0 + step, cu[b + 1])
                p = torch.arange(base + t0 - cu[b], base + t1 - cu[b], device=DEV)
                z = st["q"][t0:t1, mine].double() @ key.T / math.sqrt(dim)
                z = z.masked_fill(torch.arange(L, device=DEV) > p.view(-1, 1, 1), -math.inf)
                if kind == "sums":
                    weights[page, h, row] += torch.exp(z - st["lse"][t0:t1, mine, None].double()).sum((0, 1))
                else:
                    lse[t0:t1, mine] = torch.logsumexp(z, -1)
                    out[t0:t1, mine] = torch.exp(z - lse[t0:t1, mine, None]) @ val
    return weights if kind == "sums" else (out, lse)
