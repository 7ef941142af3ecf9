"""The paged per-head cache's operators together, as a serving loop uses them: norm, projection, keys into the pages, attention, the
weights that keys gather and eviction by them; chunks and single tokens, in captured graphs, on several streams, and in
pools larger than 32-bit offsets reach.

Tolerances are those of the operators' own tests; a run that repeats another one's work is compared bit for bit."""
import math

import pytest
import torch

from oracle import gqa
from oracle import reference as ref
from tests import _gqa
from tests.test_gpu_flash_paged_gqa import check
from tests.test_gpu_gqa_cache import check_evict, check_sums, check_write, evict, evict_case, inputs, split
from tilert_amd import kernel as K
from tilert_amd import synth
from tilert_amd.flash_paged_gqa import flash_paged_gqa
from tilert_amd.gqa_cache import gqa_cache_evict, gqa_cache_weights, gqa_cache_write
from tilert_amd.rmsnorm import add_rmsnorm_quant

pytestmark = pytest.mark.gpu
HEADS, KV, DIM, MODEL = 8, 2, 128, 2048
BF16, FP8, F32, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.float32, torch.int32


class Layer:
    """One grouped-query attention layer over a pool of pages, for caches that grow up to `total`."""

    def __init__(self, dev, total, seed, spare=12):
        pages, table, _, _, _ = _gqa.batch([1] * len(total), total, KV, DIM, spare=spare, extra_columns=1, seed=seed)
        used = set(table.flatten().tolist())
        self.free = [i for i in range(pages.shape[0]) if i not in used]
        self.dev, self.pages, self.table = dev, pages.to(dev), table.to(dev)
        g = synth.gen(seed)
        w, ws = ref.weight_quant(synth.weight_fp32((HEADS + 2 * KV) * DIM, MODEL, g))
        self.w, self.ws = w.to(dev), ws.to(dev)
        self.gamma_in = (torch.rand(MODEL, generator=g) * 0.2 + 0.9).to(dev)
        self.gq, self.gk = ((torch.rand(DIM, generator=g) * 0.2 + 0.9).to(dev) for _ in range(2))
        self.logs = torch.zeros(1, dtype=torch.uint8, device=dev)
        self.weights = torch.zeros(pages.shape[0], KV, 64, device=dev)

    def project(self, x, residual):
        rows = x.shape[0]
        total = torch.empty_like(residual)
        q, s = torch.empty(rows, MODEL, dtype=FP8, device=self.dev), torch.empty(rows, MODEL // 128, device=self.dev)
        add_rmsnorm_quant(x, residual, self.gamma_in, total, None, q, s, self.logs, model_arch="deepseek_v3_2", scale_fmt="div")
        return torch.cat([K.fp8_gemm(q[i:i + 64], s[i:i + 64], self.w, self.ws) for i in range(0, rows, 64)]).view(rows, -1, DIM)

    def step(self, joint, freqs, cu, lens):
        """Keys into the pages, attention, the weights: (queries, out, lse)."""
        q, k, v = split(joint, HEADS, KV)
        query, out = torch.full(q.shape, 7.0, dtype=BF16, device=self.dev), torch.full(q.shape, 7.0, dtype=BF16, device=self.dev)
        lse = torch.full(q.shape[:-1], 7.0, device=self.dev)
        gqa_cache_write(k, v, self.pages, self.table, cu, lens, self.gk, freqs, query=q, gamma_q=self.gq, query_out=query,
                        key_weights=self.weights)
        flash_paged_gqa(query, self.pages, self.table, cu, lens, out, lse, kv_heads=KV)
        gqa_cache_weights(query, lse, self.pages, self.table, cu, lens, self.weights)
        return query, out, lse

    def checked_step(self, joint, freqs, cu, lens):
        before, weights = self.pages.cpu(), self.weights.cpu()
        query, out, lse = self.step(joint, freqs, cu, lens)
        torch.cuda.synchronize()
        table, cu, lens = self.table.cpu(), cu.cpu(), lens.cpu()
        check_write(before, self.pages.cpu(), joint.cpu(), HEADS, KV, DIM, table, cu, lens, self.gq.cpu(), self.gk.cpu(), freqs.cpu(), False, query.cpu())
        check(self.dev, query, self.pages, table, cu, lens, KV, out, lse)
        for b, n in enumerate(lens.tolist()):  # the written keys start at 0
            for p in range(n - int(cu[b + 1] - cu[b]), n):
                weights[int(table[b, p // 64]), :, p % 64] = 0
        check_sums(self.dev, query, lse, self.pages.cpu(), table, cu, lens, KV, weights, self.weights, True)
        return query, out, lse

    def evict(self, lens, keep, recent):
        """Down to `keep` keys each: the new lengths; the sequences' old pages are free afterwards."""
        n = len(keep)
        to = torch.full((n, self.table.shape[1]), -1, dtype=I32)
        for b, m in enumerate(keep):
            for c in range(-(-(m + 3) // 64)):  # room for three more tokens
                to[b, c] = self.free.pop()
        args = (self.pages.cpu(), self.weights.cpu(), self.table.cpu(), lens.cpu(), torch.tensor(keep, dtype=I32))
        kept, slots = torch.full((n,), 77, dtype=I32, device=self.dev), torch.full((n, KV, 64 * to.shape[1]), 77, dtype=I32, device=self.dev)
        gqa_cache_evict(self.pages, self.weights, self.table, lens, args[4].to(self.dev), to.to(self.dev), kept, slots, head_dim=DIM, recent=recent)
        torch.cuda.synchronize()
        check_evict(*args, to, KV, DIM, recent, self.pages.cpu(), self.weights.cpu(), kept.cpu(), slots.cpu())
        self.table = to.to(self.dev)
        return kept


def _inputs(dev, rows, seed):
    g = torch.Generator().manual_seed(seed)
    x, r = (torch.randn(rows, MODEL, generator=g).to(BF16).to(dev) for _ in range(2))
    return x, r, inputs(rows, 1, 1, DIM, DIM, seed)[3].to(dev)


def _meta(dev, new, lens):
    return torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=I32, device=dev), torch.tensor(lens, dtype=I32, device=dev)


def test_prefill_decode_evict_decode(cuda):
    """Three prompts in two chunks, two steps of one token, an eviction by the weights so far, two more steps over what is left."""
    prompts, first = [70, 5, 200], [33, 2, 100]
    layer = Layer(cuda, [n + 2 for n in prompts], 3)
    x, r, freqs = _inputs(cuda, sum(prompts), 5)
    start = [0, 70, 75]
    for new, done in ((first, first), ([n - f for n, f in zip(prompts, first)], prompts)):
        rows = torch.cat([torch.arange(s + d - n, s + d) for s, n, d in zip(start, new, done)]).to(cuda)
        layer.checked_step(layer.project(x[rows], r[rows]), freqs[rows], *_meta(cuda, new, done))
    for step in (1, 2):
        x, r, freqs = _inputs(cuda, 3, 7 + step)
        cu, lens = _meta(cuda, [1, 1, 1], [n + step for n in prompts])
        layer.checked_step(layer.project(x, r), freqs, cu, lens)
    lens = layer.evict(lens, [40, 7, 126], recent=16)
    assert lens.tolist() == [40, 7, 126]
    for step in (1, 2, 3):
        x, r, freqs = _inputs(cuda, 3, 11 + step)
        lens = lens + 1
        layer.checked_step(layer.project(x, r), freqs, cu, lens)


def test_one_prompt_whole_and_in_pages(cuda):
    """Chunks that end where a page does give the same pages and rows, bit for bit, as the prompt at once."""
    n = 384
    whole, parts = Layer(cuda, [n], 13), Layer(cuda, [n], 13)
    x, r, freqs = _inputs(cuda, n, 15)
    joint = whole.project(x, r)
    query, out, lse = whole.step(joint, freqs, *_meta(cuda, [n], [n]))
    for a, b in ((0, 64), (64, 320), (320, 384)):
        q, o, z = parts.step(joint[a:b], freqs[a:b], *_meta(cuda, [b - a], [b]))
        assert torch.equal(q, query[a:b])
    assert torch.equal(parts.pages, whole.pages)
    check(cuda, query, whole.pages, whole.table.cpu(), torch.tensor([0, n]), torch.tensor([n]), KV, out, lse)


def _graph(run, pool=None):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool):
        out = run()
    return g, out


@pytest.mark.parametrize("total", [[300, 100], [2500, 900, 64], [20000]])  # uncut; planned and joined
def test_a_captured_decode_step(cuda, total):
    """One captured step, replayed for six tokens while the caches grow by it: the metadata is read at the replay."""
    n, steps = len(total), 6
    layer, eager = Layer(cuda, [t + steps for t in total], 11), Layer(cuda, [t + steps for t in total], 11)
    for one in (layer, eager):
        pages = one.pages.cpu()
        _gqa.fill(pages, one.table.cpu(), total, KV, DIM)
        one.pages.copy_(pages)
    cu, lens = _meta(cuda, [1] * n, total)
    x, r, freqs = _inputs(cuda, n, 13)
    joint = layer.project(x, r)
    lens += 1
    graph, got = _graph(lambda: layer.step(joint, freqs, cu, lens))
    layer.weights.zero_()
    pages = layer.pages.cpu()
    _gqa.fill(pages, layer.table.cpu(), total, KV, DIM)  # (what the run before the capture wrote, taken back)
    layer.pages.copy_(eager.pages)
    for step in range(steps):
        x, r, new_freqs = _inputs(cuda, n, 17 + step)
        joint.copy_(eager.project(x, r))
        freqs.copy_(new_freqs)
        lens.copy_(torch.tensor([t + 1 + step for t in total], dtype=I32))
        want = eager.step(joint, freqs, cu, lens)
        torch.cuda.synchronize()
        for t in got:
            t.fill_(-3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), step
        assert torch.equal(layer.pages, eager.pages) and torch.equal(layer.weights, eager.weights), step
        check(cuda, got[0], layer.pages, layer.table.cpu(), cu.cpu(), lens.cpu(), KV, got[1], got[2])


def test_a_captured_eviction(cuda):
    """Lengths, counts, weights and tables are read at the replay."""
    args = evict_case([900, 300], [500, 300], 2, 64, 61)
    dev = [t.to(cuda) for t in args]
    pages, w, table, lens, keep, to = dev
    kept, slots = torch.zeros(2, dtype=I32, device=cuda), torch.zeros(2, 2, 64 * to.shape[1], dtype=I32, device=cuda)
    graph, _ = _graph(lambda: gqa_cache_evict(pages, w, table, lens, keep, to, kept, slots, head_dim=64, recent=20))
    for i, (n, k) in enumerate((([900, 300], [500, 300]), ([610, 7], [64, 3]), ([0, 129], [3, 65]))):
        g = torch.Generator().manual_seed(i)
        case = [args[0], torch.randn(args[1].shape, generator=g), args[2].flip(1) if i == 1 else args[2],
                torch.tensor(n, dtype=I32), torch.tensor(k, dtype=I32), args[5]]
        for held, new in zip(dev, case):
            held.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        check_evict(*case, 2, 64, 20, pages.cpu(), w.cpu(), kept.cpu(), slots.cpu())


def _case(cuda, new, total, seed, heads=HEADS, kv=KV, dim=DIM, columns=9):
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, extra_columns=columns, seed=seed)
    _gqa.fill(pages, table, total, kv, dim, seed=seed)
    return _gqa.to(cuda, _gqa.queries(rows, heads, dim, seed), pages, table, cu, lens)


def _attend(case, kv=KV):
    out, lse = torch.full_like(case[0], 7.0), torch.full(case[0].shape[:-1], 7.0, device=case[0].device)
    flash_paged_gqa(*case, out, lse, kv_heads=kv)
    return out, lse


def _sums(case, lse, kv=KV):
    w = torch.zeros(case[1].shape[0], kv, 64, device=lse.device)
    gqa_cache_weights(case[0], lse, *case[1:], w)
    return w


def test_two_graphs_over_one_memory_pool(cuda):
    """Two captured calls whose workspaces lie in the same memory, replayed in turn, with eager calls between."""
    cases = [_case(cuda, [1, 1, 1], [900, 3000, 64], 19), _case(cuda, [300, 2], [700, 4000], 23)]
    want = [[t.clone() for t in _attend(c)] for c in cases]
    first, a = _graph(lambda: _attend(cases[0]))
    second, b = _graph(lambda: _attend(cases[1]), pool=first.pool())
    for i in range(4):
        for g, got, w in ((first, a, want[0]), (second, b, want[1])):
            g.replay()
            kept = [t.clone() for t in got]
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(kept, w)), i
            assert all(torch.equal(x, y) for x, y in zip(_attend(cases[i % 2]), want[i % 2]))


def test_calls_on_other_streams_at_once(cuda):
    """Four streams, each with its own calls one after another, evictions among them, while the default stream works too."""
    cases = [_case(cuda, [1] * i + [100], [500 * (i + j + 1) for j in range(i + 1)], 29 + i) for i in range(4)]
    evictions = [[t.to(cuda) for t in evict_case([700, 900], [300, 500], KV, DIM, 31 + i)] for i in range(4)]

    def work(c, e):
        out, lse = _attend(c)
        w = _sums(c, lse)
        pages, weights = e[0].clone(), e[1].clone()
        kept = torch.zeros(2, dtype=I32, device=cuda)
        gqa_cache_evict(pages, weights, *e[2:], kept, head_dim=DIM, recent=8)
        return out, lse, w, pages, weights, kept

    want = [work(c, e) for c, e in zip(cases, evictions)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[] for _ in cases]
    for _ in range(5):
        for s, c, e, g in zip(streams, cases, evictions, got):
            with torch.cuda.stream(s):
                g.append(work(c, e))
        work(cases[0], evictions[0])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for one in g for x, y in zip(one, w))


@pytest.mark.parametrize("new,total", [([1, 40], [700, 300]), ([300, 2], [400, 900])])
def test_a_pool_past_32_bit_offsets(cuda, new, total):
    """Pages just before and behind 2^31 and 2^32 bytes, and the last one of a pool of 4.9 GB."""
    size, count = gqa.page_bytes(KV, DIM), 150_000
    small, table, cu, lens, rows = _gqa.batch(new, total, KV, DIM, spare=12, seed=37)
    _gqa.fill(small, table, total, KV, DIM)
    ids = [2 ** 31 // size + i for i in (-1, 0, 1)] + [2 ** 32 // size + i for i in (-1, 0, 1)] + [count - 1]
    ids += list(range(90_000, 90_000 + small.shape[0] - len(ids)))
    where = torch.tensor(ids, dtype=torch.int64)
    pool = torch.empty(count, size, dtype=torch.uint8, device=cuda)
    pool[where.to(cuda)] = small.to(cuda)
    move = lambda t: torch.where(t >= 0, where[t.clamp_min(0).long()].to(I32), t)  # noqa: E731
    used = set(table.flatten().tolist())
    free = [i for i in range(small.shape[0]) if i not in used]
    to = torch.full((2, 3), -1, dtype=I32)
    for i in range(6):
        to[i // 3, i % 3] = free[i]
    joint, gq, gk, freqs = inputs(rows, HEADS, KV, DIM, DIM, 41)
    results = []
    for pages, tab, target in ((small.to(cuda), table, to), (pool, move(table), move(to))):
        q, k, v = split(joint.to(cuda), HEADS, KV)
        meta = _gqa.to(cuda, tab, cu, lens)
        query, weights = torch.zeros(rows, HEADS, DIM, dtype=BF16, device=cuda), torch.zeros(pages.shape[0], KV, 64, device=cuda)
        gqa_cache_write(k, v, pages, *meta, *_gqa.to(cuda, gk, freqs), query=q, gamma_q=gq.to(cuda), query_out=query, key_weights=weights)
        out, lse = _attend((query, pages, *meta))
        gqa_cache_weights(query, lse, pages, *meta, weights)
        n, slots = torch.zeros(2, dtype=I32, device=cuda), torch.zeros(2, KV, 192, dtype=I32, device=cuda)
        gqa_cache_evict(pages, weights, meta[0], meta[2], torch.tensor([150, 192], dtype=I32, device=cuda), target.to(cuda), n, slots, head_dim=DIM)
        results.append((pages, weights, query, out, lse, n, slots))
    near, far = results
    assert torch.equal(far[0][where.to(cuda)], near[0]) and torch.equal(far[1][where.to(cuda)], near[1])
    assert all(torch.equal(a, b) for a, b in zip(near[2:], far[2:])) and near[5].tolist() == [150, 192]
    check(cuda, near[2].cpu(), near[0].cpu(), table, cu, lens, KV, near[3], near[4])


@pytest.mark.parametrize("n", [64, 512, 513, 1100, 5000])
def test_many_sequences(cuda, n):
    """More sequences than one round, a launch's plan and two rounds of the search take; some are empty, some have no new token."""
    new = [(0 if i % 7 == 3 else 1 + i % 2) for i in range(n)]
    total = [max(m, (i * 37) % (900 if n <= 1100 else 90)) for i, m in enumerate(new)]
    pages, table, cu, lens, rows = _gqa.batch(new, total, 1, 64, pad=5, seed=47)
    _gqa.fill(pages, table, [t - m for m, t in zip(new, total)], 1, 64)
    joint, gq, gk, freqs = inputs(rows, 4, 1, 64, 32, 53)
    q, k, v = split(joint.to(cuda), 4, 1)
    d = _gqa.to(cuda, pages, table, cu, lens)
    query, weights = torch.full((rows, 4, 64), 7.0, dtype=BF16, device=cuda), torch.zeros(pages.shape[0], 1, 64, device=cuda)
    gqa_cache_write(k, v, *d, *_gqa.to(cuda, gk, freqs), query=q, gamma_q=gq.to(cuda), query_out=query, key_weights=weights)
    check_write(pages, d[0].cpu(), joint, 4, 1, 64, table, cu, lens, gq, gk, freqs, False, query.cpu())
    case = (query, *d)
    out, lse = _attend(case, 1)
    check(cuda, query.cpu(), d[0].cpu(), table, cu, lens, 1, out, lse)
    gqa_cache_weights(query, lse, *d, weights)
    check_sums(cuda, query, lse, d[0].cpu(), table, cu, lens, 1, torch.zeros(weights.shape), weights, True)


@pytest.mark.parametrize("n,tokens,heads,kv,dim", [(520, 3, 8, 1, 64), (520, 9, 8, 1, 128), (513, 1, 32, 2, 128), (515, 2, 40, 2, 64)])
def test_tiles_of_every_size_unplanned(cuda, n, tokens, heads, kv, dim):
    total = [tokens + i % 90 for i in range(n)]
    pages, table, cu, lens, rows = _gqa.batch([tokens] * n, total, kv, dim, seed=49)
    _gqa.fill(pages, table, total, kv, dim)
    case = _gqa.to(cuda, _gqa.queries(rows, heads, dim, 51), pages, table, cu, lens)
    out, lse = _attend(case, kv)
    check(cuda, case[0], pages, table, cu, lens, kv, out, lse)
    check_sums(cuda, case[0], lse, pages, table, cu, lens, kv, torch.zeros(pages.shape[0], kv, 64), _sums(case, lse, kv), True)


@pytest.mark.parametrize("new,total,heads,kv,dim", [
    ([12], [9000], 32, 8, 128), ([16], [300], 32, 8, 64), ([50], [700], 8, 8, 128), ([7, 9, 8], [4000, 100, 2000], 20, 4, 64),
    ([30] + [1] * 20, [60] + [200] * 20, 8, 2, 128), ([40] + [1] * 30, [4000] + [70] * 30, 4, 1, 64),
])
def test_rows_between_a_step_and_a_chunk(cuda, new, total, heads, kv, dim):
    """Tiles of 64 rows, and batches of few rows a sequence of which one has many."""
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, seed=91)
    _gqa.fill(pages, table, total, kv, dim)
    case = _gqa.to(cuda, _gqa.queries(rows, heads, dim, 93), pages, table, cu, lens)
    out, lse = _attend(case, kv)
    check(cuda, case[0], pages, table, cu, lens, kv, out, lse)
    check_sums(cuda, case[0], lse, pages, table, cu, lens, kv, torch.zeros(pages.shape[0], kv, 64), _sums(case, lse, kv), True)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("columns", [1, 60, 120, 400, 2 ** 20])
@pytest.mark.parametrize("new", [[70, 33, 1], [200, 2, 150]])
def test_the_weights_at_every_width_of_the_table(cuda, dim, columns, new):
    """The table's width decides how many pages a workgroup takes, and how many turns it has."""
    total = [900, 40, 300]
    case = _case(cuda, new, total, 95, heads=12, kv=3, dim=dim, columns=columns - 15 if columns > 15 else 0)
    out, lse = _attend(case, 3)
    check(cuda, case[0], *(t.cpu() for t in case[1:]), 3, out, lse)
    q, pages, table, cu, lens = (t.cpu() for t in case)
    check_sums(cuda, q, lse, pages, table, cu, lens, 3, torch.zeros(pages.shape[0], 3, 64), _sums(case, lse, 3), True)


@pytest.mark.parametrize("dim,heads", [(64, 1), (128, 8), (64, 100)])
def test_the_longest_cache(cuda, dim, heads):
    """2^20 pages, 2^26 keys, all of them one page, of keys that are 0 and values of 0.5, 1, 1.5 and 2: a piece's sums are exact (at
    most 2^12 pages of 64 keys in halves of a unit, 2^20), and the fewer than 2^10 that are joined add 2^-14."""
    case = list(_case(cuda, [1], [64], 97, heads=heads, kv=1, dim=dim, columns=0))
    k, v, scales = gqa.views(case[1].cpu(), 1, dim)
    page = int(case[2][0, 0])
    k[page], scales[page] = 0, 1.0
    v[page] = torch.tensor([0x30, 0x38, 0x3c, 0x40], dtype=torch.uint8)[torch.randint(0, 4, v[page].shape, generator=torch.Generator().manual_seed(98))]
    case[1] = k.new_empty(0).set_(k.untyped_storage(), 0, case[1].shape).to(cuda)
    n = 2 ** 20
    case[2] = case[2].expand(1, n).contiguous()
    case[4] = torch.full_like(case[4], n * 64)
    out, lse = _attend(case, 1)
    want = gqa.value_of(v[page, 0]).mean(-1)
    assert torch.all((out.cpu().double() - want).abs() <= (2 ** -8 + 2 ** -13) * want)
    assert torch.all((lse.cpu().double() - 26 * math.log(2)).abs() <= 2 ** -14 + 2 ** -20 * 19)


@pytest.mark.parametrize("total,keep,recent", [([70000], [65000], 10), ([140000, 66000], [70000, 64], 5000)])
def test_evictions_from_long_caches(cuda, total, keep, recent):
    """More pages than are marked at a time."""
    args = evict_case(total, keep, 1, 64, 99)
    check_evict(*args, 1, 64, recent, *evict(cuda, *args, 1, 64, recent))
    args[1].copy_(torch.randint(0, 4, args[1].shape, generator=torch.Generator().manual_seed(101)).float())  # many that are equal
    check_evict(*args, 1, 64, recent, *evict(cuda, *args, 1, 64, recent))


def test_evictions_in_the_widest_table(cuda):
    args = list(evict_case([700, 70], [300, 70], 2, 128, 103))
    wide = torch.full((2, 2 ** 20), -1, dtype=I32)
    wide[:, :args[2].shape[1]] = args[2]
    args[2] = wide
    check_evict(*args, 2, 128, 40, *evict(cuda, *args, 2, 128, 40))


def test_an_eviction_that_updates_keep_lens_in_place(cuda):
    args = evict_case([900, 300, 64], [400, 500, 64], 4, 64, 111)
    pages, w, table, lens, keep, to = (t.to(cuda) for t in args)
    slots = torch.zeros(3, 4, 64 * to.shape[1], dtype=I32, device=cuda)
    gqa_cache_evict(pages, w, table, lens, keep, to, keep, slots, head_dim=64, recent=7)
    assert keep.tolist() == [400, 300, 64]
    check_evict(*args, 4, 64, 7, pages.cpu(), w.cpu(), keep.cpu(), slots.cpu())


def test_rows_turned_in_place(cuda):
    """query_out may be the queries' own memory: a row's lanes have read it all before one of them writes."""
    joint, gq, gk, freqs = inputs(150, 8, 2, 128, 128, 113)
    pages, table, cu, lens, _ = _gqa.batch([150], [200], 2, 128, seed=115)
    q, k, v = (t.contiguous() for t in split(joint.to(cuda), 8, 2))
    args = _gqa.to(cuda, table, cu, lens, gk, freqs)
    want, out = torch.zeros_like(q), [pages.to(cuda), pages.to(cuda)]
    gqa_cache_write(k, v, out[0], *args, query=q, gamma_q=gq.to(cuda), query_out=want)
    gqa_cache_write(k, v, out[1], *args, query=q, gamma_q=gq.to(cuda), query_out=q)
    assert torch.equal(q, want) and torch.equal(out[0], out[1])


def test_weights_and_angles_that_are_aligned_to_their_elements_only(cuda):
    args = evict_case([900], [400], 2, 64, 105)
    want = evict(cuda, *args, 2, 64, 30)
    d = [t.to(cuda) for t in args]
    shifted = torch.empty(d[1].numel() + 1, device=cuda)[1:].view_as(d[1]).copy_(d[1])
    kept, slots = torch.zeros(1, dtype=I32, device=cuda), torch.zeros(1, 2, 64 * d[5].shape[1], dtype=I32, device=cuda)
    gqa_cache_evict(d[0], shifted, *d[2:], kept, slots, head_dim=64, recent=30)
    assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip((d[0], shifted, kept, slots), want))
    joint, gq, gk, freqs = inputs(70, 4, 2, 64, 64, 107)
    pages, table, cu, lens, _ = _gqa.batch([70], [70], 2, 64, seed=109)
    q, k, v = split(joint.to(cuda), 4, 2)
    results = []
    for shift in (0, 1, 3):
        move = lambda t: torch.empty(t.numel() + shift, device=cuda)[shift:].view_as(t).copy_(t)  # noqa: B023, E731
        p, out = pages.to(cuda), torch.zeros(70, 4, 64, dtype=BF16, device=cuda)
        gqa_cache_write(k, v, p, *_gqa.to(cuda, table, cu, lens), move(gk), move(freqs), query=q, gamma_q=move(gq), query_out=out)
        results.append((p, out))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(r, results[0]))


def test_a_pool_that_is_a_part_of_another(cuda):
    case = _case(cuda, [1, 20], [700, 90], 71)
    pool = torch.full((case[1].shape[0] + 7, gqa.page_bytes(KV, DIM)), 0xff, dtype=torch.uint8, device=cuda)
    pool[5:-2] = case[1]
    a, b = _attend(case), _attend((case[0], pool[5:-2], *case[2:]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("factor", [0.0, 2.0 ** -60, 2.0 ** 40])
def test_queries_of_zero_and_of_far_sizes(cuda, factor):
    """Zero and tiny queries weigh all keys alike; `scale` undoes a power of two, so that the results are the plain ones bit for bit."""
    case = _case(cuda, [1, 20], [900, 130], 79)
    q = (case[0].float() * factor).to(BF16)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:-1], 7.0, device=cuda)
    if factor > 1:
        flash_paged_gqa(q, *case[1:], out, lse, kv_heads=KV, scale=DIM ** -0.5 / factor)
        plain = _attend(case)
        assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    else:
        flash_paged_gqa(q, *case[1:], out, lse, kv_heads=KV)
        check(cuda, q, *(t.cpu() for t in case[1:]), KV, out, lse)


@pytest.mark.parametrize("new", [1, 30])
def test_sequences_that_share_pages(cuda, new):
    """A prefix in the same pages for three sequences, and a page that a sequence names twice: read, they are as any other."""
    total = [700, 800, 700]
    pages, table, cu, lens, rows = _gqa.batch([new] * 3, total, KV, DIM, seed=83)
    _gqa.fill(pages, table, total, KV, DIM)
    table[1, :9], table[2, :11] = table[0, :9], table[0, :11]
    table[2, 3] = table[2, 2]
    d = _gqa.to(cuda, _gqa.queries(rows, HEADS, DIM, 89), pages, table, cu, lens)
    check(cuda, d[0], pages, table, cu, lens, KV, *_attend(d))


@pytest.mark.parametrize("seed", range(6))
def test_metadata_that_does_not_make_sense_stays_inside(cuda, seed):
    """cu_seqlens that do not ascend, lengths and pages that are not there: what lies around the calls' tensors and the pool is left
    as it was, and a call that makes sense is right afterwards."""
    g = torch.Generator().manual_seed(100 + seed)
    B, (heads, kv, dim) = 1 + seed, [(16, 2, 64), (5, 1, 128), (40, 8, 64)][seed % 3]
    new = [1 + int(x) for x in torch.randint(0, 5 if seed < 3 else 90, (B,), generator=g)]
    total = [n + int(x) for n, x in zip(new, torch.randint(0, 1500 if seed % 2 else 200, (B,), generator=g))]
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, pad=seed % 3, seed=seed)
    _gqa.fill(pages, table, total, kv, dim)
    joint, gq, gk, freqs = inputs(rows, heads, kv, dim, 32, seed)
    q, k, v = split(joint.to(cuda), heads, kv)
    good = (q.contiguous(), *_gqa.to(cuda, pages, table, cu, lens))
    pick = lambda p, low, high, t: torch.where(torch.rand(t.shape, generator=g) < p, torch.randint(low, high, t.shape, generator=g).to(I32), t)  # noqa: E731

    def fenced(shape, dtype=F32, value=7.0):
        whole = torch.full((shape[0] + 8, *shape[1:]), value, dtype=dtype, device=cuda)
        return whole, whole[4:-4]

    for i in range(5):
        print("metadata", seed, i, flush=True)
        meta = _gqa.to(cuda, pick(0.2, -5, pages.shape[0] + 5, table), pick(0.5, -4, rows + 4, cu), pick(0.3, -50, 64 * table.shape[1] + 50, lens))
        pool, inner = fenced(pages.shape, torch.uint8, 0x55)
        inner.copy_(good[1])
        out, lse, query, w = fenced((rows, heads, dim), BF16), fenced((rows, heads)), fenced((rows, heads, dim), BF16), fenced((pages.shape[0], kv, 64))
        kept, slots = fenced((B,), I32, 7), fenced((B, kv, 128), I32, 7)
        flash_paged_gqa(good[0], inner, *meta, out[1], lse[1], kv_heads=kv)
        gqa_cache_weights(good[0], lse[1], inner, *meta, w[1])
        gqa_cache_write(k, v, inner, *meta, *_gqa.to(cuda, gk, freqs), query=q, gamma_q=gq.to(cuda), query_out=query[1], key_weights=w[1])
        keep, to = torch.randint(-4, 200, (B,), generator=g).to(I32), torch.randint(-4, pages.shape[0] + 4, (B, 2), generator=g).to(I32)
        gqa_cache_evict(inner, w[1], meta[0], meta[2], *_gqa.to(cuda, keep, to), kept[1], slots[1], head_dim=dim, recent=9 * i)
        torch.cuda.synchronize()
        for t, value in ((out[0], 7), (lse[0], 7), (query[0], 7), (w[0], 7), (kept[0], 7), (slots[0], 7), (pool, 0x55)):
            assert torch.all(t[:4] == value) and torch.all(t[-4:] == value)
    check(cuda, good[0], pages, table, cu, lens, kv, *_attend(good, kv))


@pytest.mark.parametrize("what", ["key", "value", "key scale", "value scale"])
@pytest.mark.parametrize("new,dim,back", [(3, 128, 1), (4, 64, 2), (7, 128, 3), (8, 64, 5), (15, 64, 6), (16, 64, 1)])
def test_a_bad_key_among_few_rows(cuda, what, new, dim, back):
    """Tiles of 16, 32 and 64 rows: the tokens before a key that is NaN are as without it, bit for bit, also where they share its
    page, and those from it on are NaN where the definition is; so are the weights that it gathers."""
    total = 700
    pages, table, cu, lens, rows = _gqa.batch([new], [total], 2, dim, seed=117)
    _gqa.fill(pages, table, [total], 2, dim)
    q = _gqa.queries(rows, 8, dim, 119)
    clean, clean_lse = _attend(_gqa.to(cuda, q, pages, table, cu, lens), 2)
    at = total - back
    page, row, first = int(table[0, at // 64]), at % 64, at - (total - new)
    k, v, scales = gqa.views(pages, 2, dim)
    if what == "key":
        k[page, 1, row, dim - 3] = 0xff
    elif what == "value":
        v[page, 1, dim - 5, row] = 0x7f
    else:
        scales[page, 1, 0 if what == "key scale" else 1] = math.nan
        first = max(first - row, 0)
    case = _gqa.to(cuda, q, pages, table, cu, lens)
    out, lse = _attend(case, 2)
    assert torch.equal(out[:first], clean[:first]) and torch.equal(lse[:first], clean_lse[:first])
    assert torch.equal(out[:, :4], clean[:, :4])  # the other kv head
    check(cuda, q, pages, table, cu, lens, 2, out, lse)
    assert torch.isnan(out[first:, 4:, dim - 5]).all()
    if what != "value":
        w = _sums(case, clean_lse, 2)
        check_sums(cuda, q, clean_lse, pages, table, cu, lens, 2, torch.zeros(w.shape), w, True)


@pytest.mark.parametrize("new,total,heads,kv,dim", [([3], [70], 128, 128, 64), ([40, 1], [90, 200], 128, 128, 128), ([2], [300], 126, 63, 64),
                                                    ([9], [100], 128, 16, 128), ([5, 2], [400, 30], 100, 20, 64)])
def test_up_to_128_heads(cuda, new, total, heads, kv, dim):
    pages, table, cu, lens, rows = _gqa.batch(new, total, kv, dim, seed=121)
    _gqa.fill(pages, table, total, kv, dim)
    case = _gqa.to(cuda, _gqa.queries(rows, heads, dim, 123), pages, table, cu, lens)
    out, lse = _attend(case, kv)
    check(cuda, case[0], pages, table, cu, lens, kv, out, lse)
    check_sums(cuda, case[0], lse, pages, table, cu, lens, kv, torch.zeros(pages.shape[0], kv, 64), _sums(case, lse, kv), True)
