"""GPU parity of gqa_cache_write, gqa_cache_weights and gqa_cache_evict against their definitions in 64 bits.

A norm's fp32 roundings: E = 2^-20 of a value's size bounds the mean's sum (128 terms), square root, reciprocal, two products
and the rotation's three (the size of a turned pair: the sum of both's magnitudes).  A code is within half a step of
y / scale: 2^-4 of the value, or half of e4m3's smallest step, 2^-10, times the scale."""
import math

import pytest
import torch

from oracle import gqa
from tests import _gqa
from tilert_amd.gqa_cache import gqa_cache_evict, gqa_cache_weights, gqa_cache_write

pytestmark = pytest.mark.gpu
BF16, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
E = 2.0 ** -20


def inputs(rows, heads, kv, dim, rope, seed, std=1.0):
    """q, k, v as views of a joint projection; gammas; freqs."""
    g = torch.Generator().manual_seed(seed)
    joint = (torch.randn(rows, heads + 2 * kv, dim, generator=g) * std).to(BF16)
    angle = torch.rand(rows, 1, rope // 2, generator=g, dtype=torch.float64) * 2 * math.pi
    freqs = torch.stack([angle.cos(), angle.sin()], -1).to(F32).reshape(rows, 1, rope)
    return joint, torch.rand(dim, generator=g) * 0.4 + 0.8, torch.rand(dim, generator=g) * 0.4 + 0.8, freqs


def split(joint, heads, kv):
    return joint[:, :heads], joint[:, heads:heads + kv], joint[:, heads + kv:]


def size_of(x, gamma, freqs, interleaved):
    """The size that a value's error is relative to: of a turned pair, both's magnitudes."""
    n = gqa.turned(x, gamma, None, False, 1e-6).abs()
    if freqs is None:
        return n
    ones = freqs.new_ones(freqs.shape).double().view(freqs.shape[0], 1, -1, 2)
    r = freqs.shape[-1]
    lo, hi = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    both = n[..., lo] + n[..., hi]
    out = n.clone()
    out[..., lo], out[..., hi] = both, both
    return out + 0 * ones.sum()


def check_write(before, after, joint, heads, kv, dim, table, cu, lens, gq, gk, freqs, interleaved, q_out):
    """The pages after a write against those before it."""
    q, k, v = split(joint, heads, kv)
    rows = int(cu[-1])
    want_q = gqa.turned(q[:rows], gq, None if freqs is None else freqs[:rows], interleaved, 1e-6)
    tol = 2 ** -8 * want_q.abs() + 2 * E * size_of(q[:rows], gq, None if freqs is None else freqs[:rows], interleaved)
    assert torch.all((q_out[:rows].double() - want_q).abs() <= tol)
    assert torch.all(q_out[rows:] == 7.0)
    y = torch.stack([gqa.turned(k, gk, freqs, interleaved, 1e-6), v.double()])
    size = torch.stack([size_of(k, gk, freqs, interleaved), torch.zeros_like(v, dtype=torch.float64)])
    bad = ~(torch.isfinite(y).all(-1)).all(0)  # [rows, kv]
    kc, vc, sc = gqa.views(after, kv, dim)
    ok_, ov, os_ = gqa.views(before, kv, dim)
    untouched = torch.ones(after.shape[0], dtype=torch.bool)
    for b, L in enumerate(lens.tolist()):
        n, first = int(cu[b + 1] - cu[b]), L - int(cu[b + 1] - cu[b])
        for c in range(max(first, 0) // 64, -(-L // 64)):
            lo, hi = max(first, c * 64), min(L, c * 64 + 64)
            if n == 0 or lo >= hi or c >= table.shape[1] or not 0 <= int(table[b, c]) < after.shape[0]:
                continue
            page, t0 = int(table[b, c]), int(cu[b]) + lo - first
            untouched[page] = False
            r0, r1 = lo - c * 64, hi - c * 64
            for h in range(kv):
                for i, (codes, old) in enumerate(((kc[page, h], ok_[page, h]), (vc[page, h].T, ov[page, h].T))):
                    fine = ~bad[t0:t0 + r1 - r0, h]
                    x, z = y[i, t0:t0 + r1 - r0, h], size[i, t0:t0 + r1 - r0, h]
                    amax = float(x[fine].abs().max()) if fine.any() else 0.0
                    slack = float(2 * E * z[fine].max()) if fine.any() else 0.0
                    s, s_old = float(sc[page, h, i]), float(os_[page, h, i])
                    most = gqa.scale_of(amax + slack), gqa.scale_of(max(amax - slack, 0.0))
                    if r0 and s_old > 0:
                        most = tuple(max(m, s_old) for m in most)
                    assert s in most, (s, most, s_old)
                    value = gqa.value_of(codes[r0:r1]) * s
                    off = (value - x).abs()
                    lim = torch.maximum(2 ** -4 * x.abs(), torch.tensor(2 ** -10 * s, dtype=torch.float64)) + 2 * E * z
                    assert torch.all(off[fine] <= lim[fine])
                    if i == 0:
                        assert torch.isnan(value[~fine]).all()
                    else:
                        assert torch.all(value[~fine] == 0)
                    if r0:
                        was = gqa.value_of(old[:r0]) * s_old
                        now = gqa.value_of(codes[:r0]) * s
                        if s == s_old:
                            assert torch.equal(codes[:r0], old[:r0])
                        else:
                            assert torch.equal(torch.isnan(was), torch.isnan(now))
                            seen = ~torch.isnan(was)
                            assert torch.all((was - now).abs()[seen] <= 2 ** -10 * s)
                            exact = seen & (was.abs() >= 2 ** -6 * s)
                            assert torch.equal(was[exact], now[exact])
                    assert torch.equal(codes[r1:] if i == 0 else codes[r1:][:, :0], old[r1:] if i == 0 else old[r1:][:, :0])
    assert torch.equal(after[untouched], before[untouched])


WRITES = [  # new tokens, lengths, heads, kv, dim, rope, interleaved, padding
    ([1], [1], 8, 8, 128, 128, False, 0), ([1], [64], 32, 8, 128, 64, False, 1), ([1], [65], 20, 4, 64, 64, True, 0),
    ([1], [100], 28, 4, 128, 32, True, 0), ([63], [64], 4, 1, 64, 16, False, 3), ([64], [64], 16, 2, 128, 128, False, 0),
    ([65], [70], 16, 2, 128, 128, True, 0), ([200], [200], 24, 1, 64, 32, False, 2), ([130, 1, 0, 66], [300, 7, 40, 130], 32, 8, 128, 128, False, 5),
    ([1] * 70, list(range(1, 211, 3)), 8, 2, 128, 64, False, 4), ([2, 3], [130, 66], 128, 128, 64, 64, False, 0), ([700], [1000], 3, 3, 128, 96, False, 1),
]


def write(cuda, joint, heads, kv, pages, table, cu, lens, gq, gk, freqs, **kw):
    d = joint.to(cuda)
    q, k, v = split(d, heads, kv)
    p = pages.to(cuda)
    out = torch.full((joint.shape[0], heads, joint.shape[2]), 7.0, dtype=BF16, device=cuda)
    gqa_cache_write(k, v, p, *_gqa.to(cuda, table, cu, lens, gk, freqs), query=q, gamma_q=gq.to(cuda) if gq is not None else None,
                    query_out=out, **kw)
    torch.cuda.synchronize()
    return p.cpu(), out.cpu()


@pytest.mark.parametrize("new,total,heads,kv,dim,rope,interleaved,pad", WRITES)
def test_write_against_64_bits(cuda, new, total, heads, kv, dim, rope, interleaved, pad):
    print("case", new[:8], total[:8], heads, kv, dim, flush=True)
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, pad=pad, extra_columns=1, seed=sum(total))
    _gqa.fill(pages, table, [t - n for n, t in zip(new, total)], kv, dim, std=0.7)
    joint, gq, gk, freqs = inputs(rows, heads, kv, dim, rope, 3)
    after, out = write(cuda, joint, heads, kv, pages, table, cu, lens, gq, gk, freqs, interleaved=interleaved)
    check_write(pages, after, joint, heads, kv, dim, table, cu, lens, gq, gk, freqs, interleaved, out)


@pytest.mark.parametrize("gamma,turn,std", [(True, False, 1e-7), (True, False, 1.0), (False, True, 1e-7), (False, True, 1.0), (False, True, 1e30),
                                            (False, False, 1e-7), (False, False, 1.0), (False, False, 1e30), (False, False, 3e38)])
def test_write_without_norm_or_rotation_and_sizes(cuda, gamma, turn, std):
    """Sizes from below the least scale to the largest bf16, as far as a sum of squares and a turned pair stay in fp32."""
    new, total, kv, dim = [70, 3], [100, 64], 2, 64
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, seed=5)
    _gqa.fill(pages, table, [t - n for n, t in zip(new, total)], kv, dim, std=0.01)
    joint, gq, gk, freqs = inputs(rows, 4, kv, dim, 64, 7, 0.0)
    g = torch.Generator().manual_seed(9)
    joint = ((torch.rand(joint.shape, generator=g) * 2 - 1) * std).to(BF16)
    gq, gk, freqs = gq if gamma else None, gk if gamma else None, freqs if turn else None
    after, out = write(cuda, joint, 4, kv, pages, table, cu, lens, gq, gk, freqs)
    check_write(pages, after, joint, 4, kv, dim, table, cu, lens, gq, gk, freqs, False, out)


@pytest.mark.parametrize("grow", [1.0, 2.0, 64.0, 2.0 ** 15])
def test_a_block_whose_scale_grows(cuda, grow):
    """Token by token into one page, the last ones larger: older codes move to the new scale, exactly but for subnormals."""
    kv, dim = 2, 128
    pages, table, cu, lens, _ = _gqa.batch([1], [64], kv, dim, seed=11)
    for n in (1, 2, 17, 63):
        _gqa.fill(pages, table, [n], kv, dim, std=1.0, seed=n)
        cu, lens = torch.tensor([0, 1], dtype=I32), torch.tensor([n + 1], dtype=I32)
        joint, gq, gk, freqs = inputs(1, 4, kv, dim, 128, n + 20, grow)
        after, out = write(cuda, joint, 4, kv, pages, table, cu, lens, None, None, freqs)
        check_write(pages, after, joint, 4, kv, dim, table, cu, lens, None, None, freqs, False, out)


@pytest.mark.parametrize("what", ["key nan", "key inf", "value nan", "value inf"])
def test_a_bad_token_is_nan_alone(cuda, what):
    kv, dim = 2, 128
    pages, table, cu, lens, rows = _gqa.batch([40], [90], kv, dim, seed=13)
    _gqa.fill(pages, table, [50], kv, dim)
    joint, gq, gk, freqs = inputs(rows, 4, kv, dim, 128, 15)
    joint[20, (4 if "key" in what else 6) + 1, 77] = math.nan if "nan" in what else math.inf
    after, out = write(cuda, joint, 4, kv, pages, table, cu, lens, gq, gk, freqs)
    check_write(pages, after, joint, 4, kv, dim, table, cu, lens, gq, gk, freqs, False, out)


def test_write_places_that_are_not_there(cuda):
    """Positions below 0, past the table, and pages outside the pool: nothing of the pool is written but what has a place."""
    kv, dim = 2, 64
    pages, table, cu, lens, rows = _gqa.batch([70, 70, 70, 5], [70, 200, 200, 70], kv, dim, seed=17)
    _gqa.fill(pages, table, [0, 130, 130, 65], kv, dim)
    table[1, 2], table[2, 3] = pages.shape[0], -9
    lens[0], lens[3] = 30, 64 * table.shape[1] + 2
    joint, gq, gk, freqs = inputs(rows, 4, kv, dim, 64, 19)
    after, out = write(cuda, joint, 4, kv, pages, table, cu, lens, gq, gk, freqs)
    check_write(pages, after, joint, 4, kv, dim, table, cu, lens, gq, gk, freqs, False, out)


def test_write_clears_the_weights_of_the_written_keys(cuda):
    kv, dim, new, total = 2, 64, [70, 1], [100, 65]
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, seed=21)
    _gqa.fill(pages, table, [30, 64], kv, dim)
    joint, gq, gk, freqs = inputs(rows, 4, kv, dim, 64, 23)
    w = torch.ones(pages.shape[0], kv, 64, device=cuda)
    write(cuda, joint, 4, kv, pages, table, cu, lens, gq, gk, freqs, key_weights=w)
    want = torch.ones(pages.shape[0], kv, 64)
    for b, (n, L) in enumerate(zip(new, total)):
        for p in range(L - n, L):
            want[int(table[b, p // 64]), :, p % 64] = 0
    assert torch.equal(w.cpu(), want)


def test_write_without_queries_and_repeated(cuda):
    kv, dim = 8, 128
    pages, table, cu, lens, rows = _gqa.batch([100], [230], kv, dim, seed=25)
    _gqa.fill(pages, table, [130], kv, dim)
    joint, gq, gk, freqs = inputs(rows, 16, kv, dim, 128, 27)
    want, _ = write(cuda, joint, 16, kv, pages, table, cu, lens, gq, gk, freqs)
    d, p = joint.to(cuda), pages.to(cuda)
    _, k, v = split(d, 16, kv)
    for _ in range(2):
        gqa_cache_write(k.contiguous(), v.contiguous(), p, *_gqa.to(cuda, table, cu, lens, gk, freqs))
        assert torch.equal(p.cpu(), want)


# ---------------------------------------------------------------------------------------------------- key weights
SUMS = [  # new tokens, lengths, heads, kv, dim, padding
    ([1], [1], 8, 8, 128, 0), ([1], [64], 4, 1, 64, 0), ([1], [65], 32, 8, 128, 1), ([1], [700], 28, 4, 128, 0), ([4], [300], 64, 8, 128, 0),
    ([33], [40], 10, 2, 64, 0), ([2], [500], 128, 1, 128, 0), ([64], [64], 16, 2, 128, 2), ([150], [600], 32, 8, 128, 0),
    ([1, 5, 0, 40, 1], [90, 5, 33, 400, 1], 40, 8, 128, 3), ([1] * 70, list(range(1, 211, 3)), 8, 2, 64, 4), ([300, 1], [300, 900], 8, 8, 64, 0),
]


def check_sums(cuda, q, lse, pages, table, cu, lens, kv, was, got, accumulate, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    want, tol = was.double().clone(), torch.zeros(was.shape, dtype=torch.float64)
    for page, row, w, off in gqa.key_weights(q.cpu(), lse.cpu(), pages, table, cu, lens, kv, scale):
        want[page, :, row] = w + (was[page, :, row].double() if accumulate else 0.0)
        tol[page, :, row] = off + 2.0 ** -24 * want[page, :, row].abs()
    got = got.cpu().double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = ~torch.isnan(want)
    assert torch.all((got - want).abs()[fine] <= tol[fine]), ((got - want).abs() / tol.clamp_min(1e-300))[fine].max()


@pytest.mark.parametrize("accumulate", [True, False])
@pytest.mark.parametrize("new,total,heads,kv,dim,pad", SUMS)
def test_weights_against_64_bits(cuda, new, total, heads, kv, dim, pad, accumulate):
    print("case", new[:8], total[:8], heads, kv, dim, flush=True)
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, pad=pad, extra_columns=1, seed=sum(total))
    _gqa.fill(pages, table, total, kv, dim)
    q = _gqa.queries(rows, heads, dim, 29)
    _, lse, _, _ = gqa.attention(q, pages, table, cu, lens, kv, dim ** -0.5)
    lse = lse.float()
    was = torch.rand(pages.shape[0], kv, 64, generator=torch.Generator().manual_seed(31))
    w = was.to(cuda)
    gqa_cache_weights(*_gqa.to(cuda, q, lse, pages, table, cu, lens), w, accumulate=accumulate)
    torch.cuda.synchronize()
    check_sums(cuda, q, lse, pages, table, cu, lens, kv, was, w, accumulate)
    again = was.to(cuda)
    gqa_cache_weights(*_gqa.to(cuda, q, lse, pages, table, cu, lens), again, accumulate=accumulate)
    assert torch.equal(again, w)


@pytest.mark.parametrize("new", [3, 100])
def test_weights_of_odd_places(cuda, new):
    """Rows that see nothing, bad pages, a NaN key, a table too short: only the keys that are seen change."""
    kv, dim = 2, 64
    pages, table, cu, lens, rows = _gqa.batch([new] * 4, [200, 200, 200, 200], kv, dim, seed=33)
    _gqa.fill(pages, table, [200] * 4, kv, dim)
    table[0, 1], table[1, 0], table[1, 3] = -1, pages.shape[0], -5
    lens[2], lens[3] = new // 2, 64 * table.shape[1] + 40
    gqa.views(pages, kv, dim)[0][int(table[0, 2]), 1, 9, 5] = 0x7f
    q = _gqa.queries(rows, 8, dim, 35)
    _, lse, _, _ = gqa.attention(q, pages, table, cu, lens, kv, dim ** -0.5)
    lse = torch.nan_to_num(lse.float(), nan=3.0, neginf=-math.inf)
    was = torch.rand(pages.shape[0], kv, 64, generator=torch.Generator().manual_seed(37))
    w = was.to(cuda)
    gqa_cache_weights(*_gqa.to(cuda, q, lse, pages, table, cu, lens), w)
    check_sums(cuda, q, lse, pages, table, cu, lens, kv, was, w, True)


# ------------------------------------------------------------------------------------------------------- eviction
def check_evict(pages, weights, table, lens, keep, kept_table, kv, dim, recent, after, w_after, kept_lens, slots):
    room = kept_table.shape[1] * 64
    k, v, s = gqa.views(pages, kv, dim)
    ka, va, sa = gqa.views(after, kv, dim)
    want, want_w = pages.clone(), weights.clone()
    kw, vw, sw = gqa.views(want, kv, dim)
    for b, n in enumerate(lens.tolist()):
        for h in range(kv):
            at = gqa.kept(weights, table, b, n, int(keep[b]), recent, room, pages.shape[0], h)
            assert int(kept_lens[b]) == len(at)
            assert slots[b, h].tolist() == at + [-1] * (room - len(at))
            for c in range(-(-len(at) // 64)):
                to = int(kept_table[b, c])
                if not 0 <= to < pages.shape[0]:
                    continue
                src = torch.tensor(at[64 * c:64 * c + 64])
                pg, row = table[b].long()[src // 64], src % 64
                m = len(src)
                for i, x in enumerate((gqa.value_of(k[pg, h, row]), gqa.value_of(v[pg, h, :, row]))):
                    x = x * s[pg, h, i].double()[:, None]
                    sw[to, h, i] = gqa.scale_of(float(torch.nan_to_num(x, nan=0.0).abs().max()))
                    code = (x / sw[to, h, i].double()).float().to(_gqa.FP8).view(U8)  # exact in fp32: code times a power of two
                    (kw[to, h, :m] if i == 0 else vw[to, h, :, :m].T).copy_(code)
                want_w[to, h, :m] = weights[pg, h, row]
    for got, ref in ((ka, kw), (va, vw)):
        both = (got & 0x7f == 0x7f) & (ref & 0x7f == 0x7f)  # a NaN's sign is of no account
        assert torch.equal(torch.where(both, ref, got), ref)
    assert torch.equal(sa.view(I32), sw.view(I32))
    assert torch.equal(w_after.view(I32), want_w.view(I32))


def evict(cuda, pages, weights, table, lens, keep, kept_table, kv, dim, recent):
    p, w = pages.to(cuda), weights.to(cuda)
    n = torch.full((len(lens),), 77, dtype=I32, device=cuda)
    slots = torch.full((len(lens), kv, kept_table.shape[1] * 64), 77, dtype=I32, device=cuda)
    gqa_cache_evict(p, w, *_gqa.to(cuda, table, lens, keep, kept_table), n, slots, head_dim=dim, recent=recent)
    torch.cuda.synchronize()
    return p.cpu(), w.cpu(), n.cpu(), slots.cpu()


def evict_case(total, keep, kv, dim, seed, spread=2.0):
    need = [-(-min(k, t) // 64) for k, t in zip(keep, total)]
    pages, table, _, lens, _ = _gqa.batch([0] * len(total), total, kv, dim, spare=sum(need) + 3, extra_columns=1, seed=seed)
    _gqa.fill(pages, table, total, kv, dim, spread=spread)
    used = set(table.flatten().tolist())
    free = [i for i in range(pages.shape[0]) if i not in used]
    kept_table = torch.full((len(total), max(need + [0]) + 1), -1, dtype=I32)
    for b, n in enumerate(need):
        kept_table[b, :n] = torch.tensor([free.pop() for _ in range(n)], dtype=I32)
    g = torch.Generator().manual_seed(seed + 1)
    return pages, torch.randn(pages.shape[0], kv, 64, generator=g).exp(), table, lens, torch.tensor(keep, dtype=I32), kept_table


EVICTS = [  # lengths, keys to keep, recent, kv, dim
    ([1], [1], 0, 1, 64), ([64], [1], 0, 2, 128), ([65], [64], 1, 2, 64), ([500], [250], 32, 4, 128), ([500], [250], 0, 4, 64),
    ([500], [100], 100, 2, 128), ([500], [100], 400, 2, 64), ([100], [300], 5, 8, 64), ([0, 3, 200, 64], [4, 0, 130, 64], 3, 2, 128),
    ([5000], [1777], 64, 2, 64), ([30, 2000, 700], [10, 1000, 699], 8, 3, 128), ([20000], [100], 10, 1, 64), ([-3, 70], [5, -2], 2, 2, 64),
]


@pytest.mark.parametrize("total,keep,recent,kv,dim", EVICTS)
def test_evict_against_the_definition(cuda, total, keep, recent, kv, dim):
    print("case", total, keep, recent, kv, dim, flush=True)
    args = evict_case([max(t, 0) for t in total], [max(k, 0) for k in keep], kv, dim, sum(total))
    args[3].copy_(torch.tensor(total)), args[4].copy_(torch.tensor(keep))
    check_evict(*args, kv, dim, recent, *evict(cuda, *args, kv, dim, recent))


@pytest.mark.parametrize("what", ["equal", "few values", "zeros", "nan", "infinite", "negative"])
def test_weights_that_tie_and_odd_ones(cuda, what):
    args = evict_case([900, 70], [333, 20], 2, 64, 41)
    w = args[1]
    g = torch.Generator().manual_seed(43)
    if what == "equal":
        w.fill_(0.25)
    elif what == "few values":
        w.copy_(torch.randint(0, 3, w.shape, generator=g).float())
    elif what == "zeros":
        w.copy_(torch.where(torch.rand(w.shape, generator=g) < 0.5, 0.0, -0.0))
    else:
        some = torch.rand(w.shape, generator=g) < 0.2
        w[some] = {"nan": math.nan, "infinite": math.inf, "negative": -1.0}[what]
        if what == "infinite":
            w[torch.rand(w.shape, generator=g) < 0.2] = -math.inf
    check_evict(*args, 2, 64, 16, *evict(cuda, *args, 2, 64, 16))


def test_evict_keeps_nan_keys_and_bad_pages_out(cuda):
    """A NaN key stays NaN, keys of pages outside the pool are not there, and places outside it are dropped."""
    args = evict_case([700, 700], [300, 500], 2, 128, 47)
    pages, w, table, lens, keep, kept_table = args
    gqa.views(pages, 2, 128)[0][int(table[0, 3]), 1, 7] = 0x7f
    w[int(table[0, 3]), 1, 7] = 1e9
    table[0, 1], table[1, 10], table[1, 0] = -1, pages.shape[0], -2 ** 31
    kept_table[0, 2], kept_table[1, 0] = -4, pages.shape[0] + 3
    check_evict(*args, 2, 128, 40, *evict(cuda, *args, 2, 128, 40))
    args[4][1] = 690  # more than there are
    check_evict(*args, 2, 128, 40, *evict(cuda, *args, 2, 128, 40))


def test_evict_into_a_table_that_is_too_short(cuda):
    args = list(evict_case([700], [400], 2, 64, 53))
    args[5] = args[5][:, :3].contiguous()
    check_evict(*args, 2, 64, 500, *evict(cuda, *args, 2, 64, 500))
    check_evict(*args, 2, 64, 5, *evict(cuda, *args, 2, 64, 5))
