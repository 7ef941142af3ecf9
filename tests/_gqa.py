"""Batches over the paged per-head cache for tests: pages in random order, what holds no key filled with 0xff (NaN codes, NaN
scales), so that whatever reads it shows it."""
import torch

from oracle import gqa

BF16, F32, I32, FP8, U8 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn, torch.uint8


def batch(new, total, kv, dim, *, pad=0, spare=3, extra_columns=0, seed=0):
    """CPU tensors: (pages, table, cu, lens, rows) for sequences of `new` tokens in caches of `total` keys."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-t // gqa.KEYS) for t in total]
    order = torch.randperm(sum(need) + spare, generator=g).to(I32)
    table = torch.full((len(new), max(need + [0]) + extra_columns or 1), -1, dtype=I32)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = order[first:first + n]
        first += n
    pages = torch.full((order.numel(), gqa.page_bytes(kv, dim)), 0xff, dtype=U8)
    cu = torch.tensor([0, *torch.tensor(new, dtype=torch.int64).cumsum(0).tolist()], dtype=I32)
    return pages, table, cu, torch.tensor(total, dtype=I32), int(cu[-1]) + pad


def codes_of(x, scale):
    return (x / scale).clamp(-448, 448).to(FP8).view(U8)


def fill(pages, table, total, kv, dim, seed=1, std=1.0, spread=0.0):
    """Keys and values of N(0, std) for every sequence's positions, in place; `spread`: the blocks' own sizes, as a power of two."""
    g = torch.Generator().manual_seed(seed)
    k, v, scales = gqa.views(pages, kv, dim)
    for b, n in enumerate(total):
        for c in range(-(-n // gqa.KEYS)):
            page, rows = int(table[b, c]), min(gqa.KEYS, n - c * gqa.KEYS)
            x = torch.randn(2, kv, rows, dim, generator=g) * std * torch.exp2(spread * torch.randn(2, kv, 1, 1, generator=g))
            for h in range(kv):
                for i in range(2):
                    scales[page, h, i] = gqa.scale_of(float(x[i, h].abs().max()))
                k[page, h, :rows] = codes_of(x[0, h], scales[page, h, 0])
                v[page, h, :, :rows] = codes_of(x[1, h], scales[page, h, 1]).T


def queries(rows, heads, dim, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, heads, dim, generator=g) * std).to(BF16)


def to(dev, *ts):
    return tuple(t.to(dev) if t is not None else None for t in ts)
