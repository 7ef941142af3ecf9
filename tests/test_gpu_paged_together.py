"""The paged cache's operators together, as a serving loop uses them: norm, projection, keys into the pages, attention;
chunks and single tokens, in captured graphs, on several streams, and in pools larger than 32-bit offsets reach.

Tolerances are those of the operators' own tests; a run that repeats another one's work is compared bit for bit."""
import pytest
import torch

from oracle import paged
from oracle import reference as ref
from tests import _paged
from tests._tol import assert_gemm_close
from tests.test_gpu_flash_paged_mla import check, queries
from tests.test_gpu_mla_cache import E, _inputs
from tilert_amd import kernel as K
from tilert_amd import synth
from tilert_amd.flash_paged_mla import flash_paged_mla
from tilert_amd.flash_sparse_mla import flash_sparse_mla, softmax_scale
from tilert_amd.mla_cache import mla_cache_read, mla_cache_write
from tilert_amd.rmsnorm import add_rmsnorm_quant

pytestmark = pytest.mark.gpu
ARCH, HEADS, DIM = "deepseek_v3_2", 16, 2048
BF16, FP8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int32


class Layer:
    """The key half of one attention layer over a pool of pages, for caches that grow up to `total`."""

    def __init__(self, dev, total, seed):
        pages, table, _, _, _ = _paged.batch([1] * len(total), total, extra_columns=1, seed=seed)
        self.dev, self.pages, self.table = dev, pages.to(dev), table.to(dev)
        g = synth.gen(seed)
        w, ws = ref.weight_quant(synth.weight_fp32(576, DIM, g))
        self.w, self.ws = w.to(dev), ws.to(dev)
        self.gamma_in = (torch.rand(DIM, generator=g) * 0.2 + 0.9).to(dev)
        self.gamma = (torch.rand(512, generator=g) * 0.2 + 0.9).to(dev)
        self.logs = torch.zeros(1, dtype=torch.uint8, device=dev)

    def keys(self, x, residual, freqs, cu, lens):
        """One step's keys: (the residual sum, the keys before their norm)."""
        rows = x.shape[0]
        total = torch.empty_like(residual)
        q, s = torch.empty(rows, DIM, dtype=FP8, device=self.dev), torch.empty(rows, DIM // 128, device=self.dev)
        add_rmsnorm_quant(x, residual, self.gamma_in, total, None, q, s, self.logs, model_arch=ARCH, scale_fmt="div")
        both = torch.cat([K.fp8_gemm(q[i:i + 64], s[i:i + 64], self.w, self.ws) for i in range(0, rows, 64)])
        kv, pe = both[:, :512].contiguous(), both[:, 512:].contiguous()
        mla_cache_write(kv, pe, self.pages, self.table, cu, lens, self.gamma, freqs)
        return total, kv

    def attend(self, q, qp, cu, lens):
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:-1], 7.0, device=self.dev)
        flash_paged_mla(q, qp, self.pages, self.table, cu, lens, out, lse, model_arch=ARCH)
        return out, lse


def _step_inputs(dev, rows, seed):
    g = torch.Generator().manual_seed(seed)
    x, r = (torch.randn(rows, DIM, generator=g).to(BF16).to(dev) for _ in range(2))
    return (x, r, _inputs(rows, seed)[3].to(dev), *(t.to(dev) for t in queries(rows, HEADS, seed)))


def _meta(dev, new, lens):
    return torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=I32, device=dev), torch.tensor(lens, dtype=I32, device=dev)


def test_prefill_in_chunks_then_decode(cuda):
    """Three prompts, once at a time and once in two chunks, then two steps of one token: the pages are equal, every
    attention is right over them, the keys are their projections', and the flat form serves the sparse operator."""
    prompts, steps = [70, 5, 200], 2
    total = [n + steps for n in prompts]
    whole, parts = Layer(cuda, total, 3), Layer(cuda, total, 3)
    x, r, freqs, q, qp = _step_inputs(cuda, sum(prompts), 5)
    cu, lens = _meta(cuda, prompts, prompts)
    residual, kv = whole.keys(x, r, freqs, cu, lens)
    out, lse = whole.attend(q, qp, cu, lens)
    check(cuda, q, qp, whole.pages, whole.table, cu, lens, out, lse)
    assert torch.equal(residual, (x.float() + r.float()).to(BF16))
    n = paged.norm(kv, whole.gamma, 1e-6)
    codes, scales, _ = paged.views(whole.pages)
    for t, page, row in paged.places(whole.pages.shape[0], whole.table, cu, lens, sum(prompts)):
        s = scales[page, row].double()
        off = (codes[page, row].double() * s - n[t]).abs()
        assert torch.all(off <= torch.maximum(2 ** -4 * n[t].abs(), 2 ** -10 * s) + 2 * E * n[t].abs())

    first = [n // 2 for n in prompts]
    start = [0, 70, 75]
    for new, done in ((first, first), ([n - f for n, f in zip(prompts, first)], prompts)):
        rows = torch.cat([torch.arange(s + d - n, s + d) for s, n, d in zip(start, new, done)]).to(cuda)
        c, ln = _meta(cuda, new, done)
        parts.keys(x[rows], r[rows], freqs[rows], c, ln)
        o, z = parts.attend(q[rows], qp[rows], c, ln)
        check(cuda, q[rows], qp[rows], parts.pages, parts.table, c, ln, o, z)
    assert torch.equal(parts.pages, whole.pages)

    for step in range(1, steps + 1):
        x, r, freqs, q, qp = _step_inputs(cuda, 3, 7 + step)
        cu, lens = _meta(cuda, [1, 1, 1], [n + step for n in prompts])
        whole.keys(x, r, freqs, cu, lens)
        out, lse = whole.attend(q, qp, cu, lens)
        check(cuda, q, qp, whole.pages, whole.table, cu, lens, out, lse)

    cu, lens = _meta(cuda, total, total)
    flat, pe = torch.zeros(sum(total), 512, dtype=BF16, device=cuda), torch.zeros(sum(total), 64, dtype=BF16, device=cuda)
    mla_cache_read(whole.pages, whole.table, cu, lens, flat, pe)
    at = 0
    for b, n in enumerate(total):
        idx = torch.arange(n, dtype=I32, device=cuda)[None, None]
        sparse = torch.zeros(1, 1, HEADS, 512, dtype=BF16, device=cuda)
        flash_sparse_mla(q[b][None, None], qp[b][None, None], flat[None, at:at + n], pe[None, at:at + n], idx,
                         torch.tensor([n - 1], dtype=I32, device=cuda), sparse, None, model_arch=ARCH)
        want = ref.flash_sparse_mla(q[b][None].cpu(), qp[b][None].cpu(), flat[at:at + n].cpu(), pe[at:at + n].cpu(), idx[0].cpu(),
                                    n - 1, softmax_scale(ARCH))
        assert_gemm_close(sparse[0], want, "the sparse operator over the flat keys")
        at += n


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


@pytest.mark.parametrize("total", [[300, 100], [2500, 900, 64]])  # one kernel; split and joined
def test_a_captured_decode_step(cuda, total):
    """One captured step, replayed for six tokens while the caches grow by it: the metadata is read at the replay."""
    n, steps = len(total), 6
    layer, eager = Layer(cuda, [t + steps for t in total], 11), Layer(cuda, [t + steps for t in total], 11)
    for one in (layer, eager):
        pages = one.pages.cpu()
        _paged.fill(pages, one.table.cpu(), total)
        one.pages.copy_(pages)
    cu, lens = _meta(cuda, [1] * n, total)
    held = _step_inputs(cuda, n, 13)
    x, r, freqs, q, qp = held
    lens += 1
    graph, (residual, out, lse) = _graph(lambda: (layer.keys(x, r, freqs, cu, lens)[0], *layer.attend(q, qp, cu, lens)))
    for step in range(steps):
        new = _step_inputs(cuda, n, 17 + step)
        for a, b in zip(held, new):
            a.copy_(b)
        lens.copy_(torch.tensor([t + 1 + step for t in total], dtype=I32))
        want_residual = eager.keys(new[0], new[1], new[2], cu, lens)[0]
        want = eager.attend(new[3], new[4], cu, lens)
        torch.cuda.synchronize()
        for t in (residual, out, lse):
            t.fill_(-3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(residual, want_residual) and torch.equal(out, want[0]) and torch.equal(lse, want[1]), step
        assert torch.equal(layer.pages, eager.pages), step
        check(cuda, new[3], new[4], layer.pages, layer.table, cu, lens, out, lse)


def _attention_case(cuda, new, total, seed):
    pages, table, cu, lens, rows = _paged.batch(new, total, extra_columns=9, seed=seed)
    _paged.fill(pages, table, total, seed=seed)
    return _paged.to(cuda, *queries(rows, HEADS, seed), pages, table, cu, lens)


def _attend(case):
    out, lse = torch.full_like(case[0], 7.0), torch.full(case[0].shape[:-1], 7.0, device=case[0].device)
    flash_paged_mla(*case, out, lse, model_arch=ARCH)
    return out, lse


def test_two_graphs_over_one_memory_pool(cuda):
    """Two captured calls whose workspaces lie in the same memory, replayed in turn, with eager calls between."""
    cases = [_attention_case(cuda, [1, 1, 1], [900, 3000, 64], 19), _attention_case(cuda, [30, 2], [700, 4000], 23)]
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
    """Four streams, each with its own call after call, while the default stream works too."""
    cases = [_attention_case(cuda, [1] * (i + 1), [500 * (i + j + 1) for j in range(i + 1)], 29 + i) for i in range(4)]
    want = [[t.clone() for t in _attend(c)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(6):
        for s, c, g in zip(streams, cases, got):
            with torch.cuda.stream(s):
                g.append(_attend(c))
        _attend(cases[0])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, y) for pair in g for x, y in zip(pair, w))


@pytest.mark.parametrize("new,total", [([1, 40], [700, 300])])
def test_a_pool_past_32_bit_offsets(cuda, new, total):
    """Pages just before and behind 2^31 and 2^32 bytes, and the last one of a pool of 4.5 GB."""
    small, table, cu, lens, rows = _paged.batch(new, total, seed=37)
    _paged.fill(small, table, total)
    ids = [2 ** 31 // 41216 + i for i in (-1, 0, 1)] + [2 ** 32 // 41216 + i for i in (-1, 0, 1)] + [109_999]
    ids += list(range(60_000, 60_000 + small.shape[0] - len(ids)))
    where = torch.tensor(ids, dtype=torch.int64)
    pool = torch.empty(110_000, paged.PAGE_BYTES, dtype=torch.uint8, device=cuda)
    pool[where.to(cuda)] = small.to(cuda)
    far = torch.where(table >= 0, where[table.clamp_min(0).long()].to(I32), table)
    q, qp = queries(rows, HEADS, 41)
    near = _paged.to(cuda, q, qp, small, table, cu, lens)
    away = (near[0], near[1], pool, far.to(cuda), near[4], near[5])
    kv, pe, gamma, freqs = _inputs(rows, 43)
    for c in (near, away):
        mla_cache_write(*_paged.to(cuda, kv, pe), c[2], c[3], c[4], c[5], gamma.to(cuda), freqs.to(cuda))
    assert torch.equal(pool[where.to(cuda)], near[2])
    a, b = _attend(near), _attend(away)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    check(cuda, q, qp, near[2], table, cu, lens, *a)
    flat = [torch.zeros(rows, n, dtype=BF16, device=cuda) for n in (512, 64, 512, 64)]
    mla_cache_read(*near[2:], flat[0], flat[1])
    mla_cache_read(*away[2:], flat[2], flat[3])
    assert torch.equal(flat[0], flat[2]) and torch.equal(flat[1], flat[3]) and flat[0].any()


@pytest.mark.parametrize("n", [64, 600, 1100, 2100, 5000])
def test_many_sequences(cuda, n):
    """More sequences than one round, one pass, a split launch's plan and two rounds of the search take; some are
    empty, some have no new token."""
    new = [(0 if i % 7 == 3 else 1 + i % 2) for i in range(n)]
    total = [max(m, (i * 37) % (700 if n <= 1100 else 90)) for i, m in enumerate(new)]
    pages, table, cu, lens, rows = _paged.batch(new, total, pad=5, seed=47)
    _paged.fill(pages, table, total)
    kv, pe, gamma, _ = _inputs(rows, 53)
    d = _paged.to(cuda, *queries(rows, 8, 59), pages, table, cu, lens)
    mla_cache_write(kv.to(cuda), pe.to(cuda), *d[2:], gamma.to(cuda))
    out, lse = _attend(d)
    codes, scales, rope = paged.views(d[2].cpu())
    where = torch.tensor(paged.places(pages.shape[0], table, cu, lens, rows))
    s = scales[where[:, 1], where[:, 2]].double()[:, None]
    got = codes.view(torch.uint8)[where[:, 1], where[:, 2]].view(FP8).double() * s
    want = paged.norm(kv, gamma, 1e-6)[where[:, 0]]
    assert torch.all((got - want).abs() <= torch.maximum(2 ** -4 * want.abs(), 2 ** -10 * s) + 2 * E * want.abs())
    assert torch.equal(rope[where[:, 1], where[:, 2]], pe[where[:, 0]])
    check(cuda, d[0], d[1], d[2], table, cu, lens, out, lse)
    flat, flat_pe = torch.full((rows, 512), 7.0, dtype=BF16, device=cuda), torch.full((rows, 64), 7.0, dtype=BF16, device=cuda)
    mla_cache_read(*d[2:], flat, flat_pe)
    assert torch.equal(flat_pe[where[:, 0].to(cuda)].cpu(), pe[where[:, 0]]) and torch.all(flat[int(cu[-1]):] == 7.0)


@pytest.mark.parametrize("new", [640, 1100])
def test_more_row_tiles_than_a_split_launch_plans(cuda, new):
    """Many tiles over a long table: planned, and one workgroup a tile."""
    pages, table, cu, lens, rows = _paged.batch([new, 1], [new + 60, 3], seed=61)
    _paged.fill(pages, table, [new + 60, 3])
    d = _paged.to(cuda, *queries(rows, 128, 67), pages, table, cu, lens)
    check(cuda, *d[:4], cu, lens, *_attend(d))


def test_a_pool_that_is_a_part_of_another(cuda):
    case = _attention_case(cuda, [1, 20], [700, 90], 71)
    pool = torch.full((case[2].shape[0] + 7, paged.PAGE_BYTES), 0xff, dtype=torch.uint8, device=cuda)
    pool[5:-2] = case[2]
    a, b = _attend(case), _attend((*case[:2], pool[5:-2], *case[3:]))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new,total", [([1], [200]), ([40, 1], [90, 3000])])
def test_a_bad_query_row_touches_no_other(cuda, value, new, total):
    case = _attention_case(cuda, new, total, 73)
    clean = _attend(case)
    q, qp = case[0].clone(), case[1].clone()
    q[0, 3, 100], qp[0, 5, 7], q[-1, 1, 0] = value, value, value
    out, lse = _attend((q, qp, *case[2:]))
    bad = torch.zeros(out.shape[:2], dtype=torch.bool, device=cuda)
    bad[0, 3] = bad[0, 5] = bad[-1, 1] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.equal(out[~bad], clean[0][~bad]) and torch.equal(lse[~bad], clean[1][~bad])


@pytest.mark.parametrize("factor", [0.0, 2.0 ** -60, 2.0 ** 40])
def test_queries_of_zero_and_of_far_sizes(cuda, factor):
    """Zero and tiny queries weigh all keys alike; for huge ones one key is left.  The factor is a power of two and
    `scale` undoes it for the huge ones, so that the results are the plain ones bit for bit."""
    case = _attention_case(cuda, [1, 20], [900, 130], 79)
    q, qp = (case[0].float() * factor).to(BF16), (case[1].float() * factor).to(BF16)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:-1], 7.0, device=cuda)
    if factor > 1:
        base = softmax_scale(ARCH)
        flash_paged_mla(q, qp, *case[2:], out, lse, model_arch=ARCH, scale=base / factor)
        plain = _attend(case)
        assert torch.equal(out, plain[0]) and torch.equal(lse, plain[1])
    else:
        flash_paged_mla(q, qp, *case[2:], out, lse, model_arch=ARCH)
        check(cuda, q, qp, *(t.cpu() for t in case[2:]), out, lse)


@pytest.mark.parametrize("seed", range(6))
def test_metadata_that_does_not_make_sense_stays_inside(cuda, seed):
    """cu_seqlens that do not ascend, lengths and pages that are not there, in both forms of the launch: what lies around
    the call's tensors and the pool is left as it was, and a call that makes sense is right afterwards."""
    g = torch.Generator().manual_seed(100 + seed)
    B, heads = 1 + seed, (16, 5, 40)[seed % 3]
    new = [1 + int(x) for x in torch.randint(0, 5, (B,), generator=g)]
    total = [n + int(x) for n, x in zip(new, torch.randint(0, 900 if seed % 2 else 200, (B,), generator=g))]
    pages, table, cu, lens, rows = _paged.batch(new, total, pad=seed % 3, seed=seed)
    _paged.fill(pages, table, total)
    good = _paged.to(cuda, *queries(rows, heads, seed), pages, table, cu, lens)
    for _ in range(5):
        bad_cu = torch.where(torch.rand(B + 1, generator=g) < 0.5, torch.randint(-4, rows + 4, (B + 1,), generator=g).to(I32), cu)
        bad_lens = torch.where(torch.rand(B, generator=g) < 0.3, torch.randint(-50, 64 * table.shape[1] + 50, (B,), generator=g).to(I32), lens)
        bad_table = torch.where(torch.rand(table.shape, generator=g) < 0.2, torch.randint(-5, pages.shape[0] + 5, table.shape, generator=g).to(I32), table)
        pool = torch.full((pages.shape[0] + 4, paged.PAGE_BYTES), 0x55, dtype=torch.uint8, device=cuda)
        pool[2:-2] = good[2]
        out = torch.full((rows + 8, heads, 512), 7.0, dtype=BF16, device=cuda)
        lse = torch.full((rows + 8, heads), 7.0, device=cuda)
        flat, flat_pe = torch.full((rows + 8, 512), 7.0, dtype=BF16, device=cuda), torch.full((rows + 8, 64), 7.0, dtype=BF16, device=cuda)
        meta = _paged.to(cuda, bad_table, bad_cu, bad_lens)
        flash_paged_mla(good[0], good[1], pool[2:-2], *meta, out[4:-4], lse[4:-4], model_arch=ARCH)
        mla_cache_read(pool[2:-2], *meta, flat[4:-4], flat_pe[4:-4])
        kv, pe, gamma, _ = _inputs(rows, seed)
        mla_cache_write(*_paged.to(cuda, kv, pe), pool[2:-2], *meta, gamma.to(cuda))
        torch.cuda.synchronize()
        for t in (out, lse, flat, flat_pe):
            assert torch.all(t[:4] == 7.0) and torch.all(t[-4:] == 7.0)
        assert torch.all(pool[:2] == 0x55) and torch.all(pool[-2:] == 0x55)
    check(cuda, *good[:4], cu, lens, *_attend(good))


@pytest.mark.parametrize("new", [1, 30])
def test_sequences_that_share_pages(cuda, new):
    """A prefix in the same pages for three sequences, and a page that a sequence names twice."""
    total = [700, 800, 700]
    pages, table, cu, lens, rows = _paged.batch([new] * 3, total, seed=83)
    _paged.fill(pages, table, total)
    table[1, :9], table[2, :11] = table[0, :9], table[0, :11]
    table[2, 3] = table[2, 2]
    d = _paged.to(cuda, *queries(rows, HEADS, 89), pages, table, cu, lens)
    check(cuda, *d[:4], cu, lens, *_attend(d))
    flat, pe = torch.zeros(sum(total), 512, dtype=BF16, device=cuda), torch.zeros(sum(total), 64, dtype=BF16, device=cuda)
    mla_cache_read(d[2], d[3], *_meta(cuda, total, total), flat, pe)
    assert torch.equal(flat[:64 * 9], flat[700:700 + 64 * 9]) and torch.equal(flat[1500 + 128:1500 + 192], flat[1500 + 192:1500 + 256])
