"""Batches over the paged latent cache for tests: pages in random order, rows of no key filled with 0xff (NaN codes, NaN
scales, NaN rope parts), so that whatever reads one shows it."""
import torch

from oracle import paged

BF16, F32, FP8 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def batch(new, total, *, pad=0, spare=3, extra_columns=0, seed=0):
    """CPU tensors: (pages, table, cu, lens, rows) for sequences of `new` tokens in caches of `total` keys."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-t // paged.KEYS) for t in total]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(new), max(need + [0]) + extra_columns or 1), -1, dtype=torch.int32)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = order[first:first + n]
        first += n
    pages = torch.full((order.numel(), paged.PAGE_BYTES), 0xff, dtype=torch.uint8)
    cu = torch.tensor([0, *torch.tensor(new, dtype=torch.int64).cumsum(0).tolist()], dtype=torch.int32)
    return pages, table, cu, torch.tensor(total, dtype=torch.int32), int(cu[-1]) + pad


def fill(pages, table, total, seed=1, std=1.0):
    """Keys of N(0, std) latents for every sequence's positions, quantised per key, in place."""
    g = torch.Generator().manual_seed(seed)
    codes, scales, rope = paged.views(pages)
    for b, n in enumerate(total):
        p = torch.arange(n)
        page, row = table[b].long()[p // paged.KEYS], p % paged.KEYS
        v = torch.randn(n, paged.LATENT, generator=g) * std
        s = v.abs().amax(-1).clamp_min(1e-4) / 448 if n else v.new_zeros(0)
        codes.view(torch.uint8)[page, row] = (v / s[:, None]).clamp(-448, 448).to(FP8).view(torch.uint8)
        scales[page, row] = s
        rope[page, row] = torch.randn(n, paged.ROPE, generator=g).to(BF16)


def to(dev, *ts):
    return tuple(t.to(dev) if t is not None else None for t in ts)
