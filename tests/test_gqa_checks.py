"""Refusals of the paged per-head cache's operators: the wrappers' and the C entries' argument checks, which need no GPU; the page
layout that the oracle reads."""
import pytest
import torch

from oracle import gqa
from tests import _gqa
from tests.test_paged_checks import BATCH_C, P, _refused
from tilert_amd import _lib
from tilert_amd.flash_paged_gqa import flash_paged_gqa
from tilert_amd.gqa_cache import gqa_cache_evict, gqa_cache_weights, gqa_cache_write, gqa_page_bytes

BF16, F32, I32 = torch.bfloat16, torch.float32, torch.int32
HEADS, KV, DIM = 8, 2, 64


def _args(**changes):
    """Arguments that pass every check but that of the device."""
    pages, table, cu, lens, rows = _gqa.batch([2, 3], [70, 3], KV, DIM)
    a = dict(q=torch.zeros(rows, HEADS, DIM, dtype=BF16), k=torch.zeros(rows, KV, DIM, dtype=BF16), v=torch.zeros(rows, KV, DIM, dtype=BF16),
             pages=pages, table=table, cu=cu, lens=lens, out=torch.zeros(rows, HEADS, DIM, dtype=BF16), lse=torch.zeros(rows, HEADS),
             gk=torch.ones(DIM), gq=torch.ones(DIM), freqs=torch.zeros(rows, 1, DIM), w=torch.zeros(pages.shape[0], KV, 64),
             keep=torch.ones(2, dtype=I32), to=torch.full((2, 3), 1, dtype=I32), kept=torch.zeros(2, dtype=I32),
             slots=torch.zeros(2, KV, 192, dtype=I32), dim=DIM, kv=KV)
    for name, f in changes.items():
        a[name] = f(a[name])
    return a


def _attend(a, **kw):
    flash_paged_gqa(a["q"], a["pages"], a["table"], a["cu"], a["lens"], a["out"], a["lse"], kv_heads=a["kv"], **kw)


def _write(a, **kw):
    gqa_cache_write(a["k"], a["v"], a["pages"], a["table"], a["cu"], a["lens"], a["gk"], a["freqs"],
                    **{"query": a["q"], "gamma_q": a["gq"], "query_out": a["out"], "key_weights": a["w"], **kw})


def _sum(a, **kw):
    gqa_cache_weights(a["q"], a["lse"], a["pages"], a["table"], a["cu"], a["lens"], a["w"], **kw)


def _evict(a, **kw):
    gqa_cache_evict(a["pages"], a["w"], a["table"], a["lens"], a["keep"], a["to"], a["kept"], a["slots"], head_dim=a["dim"], **kw)


ALL = [_attend, _write, _sum, _evict]


@pytest.mark.parametrize("op", ALL)
def test_tensors_off_the_gpu(op):
    with pytest.raises(ValueError, match="GPU"):
        op(_args())


@pytest.mark.parametrize("change,text", [
    (dict(pages=lambda t: t.to(torch.int8)), "contiguous uint8"), (dict(pages=lambda t: t[:, :-128]), "contiguous uint8"),
    (dict(pages=lambda t: t[::2]), "contiguous uint8"), (dict(pages=lambda t: t.flatten()), "contiguous uint8"),
    (dict(table=lambda t: t.long()), "int32"), (dict(lens=lambda t: t.float()), "int32"), (dict(table=lambda t: t.T), "contiguous"),
    (dict(table=lambda t: t[0]), "max_pages"), (dict(lens=lambda t: t[:1]), "seq_lens"), (dict(lens=lambda t: torch.cat([t, t])[::2]), "contiguous"),
])
@pytest.mark.parametrize("op", ALL)
def test_a_pool_or_table_that_is_none(op, change, text):
    with pytest.raises(ValueError, match=text):
        op(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(cu=lambda t: t.long()), "int32"), (dict(cu=lambda t: t[:-1]), "cu_seqlens"), (dict(cu=lambda t: torch.cat([t, t])[::2]), "contiguous"),
])
@pytest.mark.parametrize("op", [_attend, _write, _sum])
def test_ranges_that_are_none(op, change, text):
    with pytest.raises(ValueError, match=text):
        op(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(q=lambda t: t.half()), "bfloat16"), (dict(q=lambda t: t[:, 0]), "bfloat16"), (dict(q=lambda t: t[..., :32]), "head_dim|contiguous|query is"),
    (dict(q=lambda t: t[..., ::2]), "head_dim|contiguous|query is"), (dict(q=lambda t: t.transpose(0, 1)), "contiguous|heads|query"),
    (dict(q=lambda t: torch.zeros(5, HEADS, DIM + 3, dtype=BF16)[..., :DIM]), "contiguous"),
    (dict(q=lambda t: torch.zeros(5, HEADS * DIM + 4, dtype=BF16)[:, :HEADS * DIM].unflatten(1, (HEADS, DIM))), "multiple of 8"),
    (dict(q=lambda t: t[:1].expand(5, -1, -1)), "contiguous"), (dict(q=lambda t: t[:, :7]), "heads"),
])
@pytest.mark.parametrize("op", [_attend, _write, _sum])
def test_queries_that_do_not_fit(op, change, text):
    with pytest.raises(ValueError, match=text):
        op(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(out=lambda t: t.float()), "output"), (dict(out=lambda t: t[:1]), "output"), (dict(out=lambda t: torch.zeros(5, DIM, HEADS, dtype=BF16).transpose(1, 2)), "output"),
    (dict(lse=lambda t: t.double()), "lse"), (dict(lse=lambda t: t[:1]), "lse"), (dict(lse=lambda t: torch.zeros(HEADS, 5).T), "lse"),
    (dict(kv=lambda n: 0), "kv_heads"), (dict(kv=lambda n: 129), "kv_heads"), (dict(kv=lambda n: 3), "kv_pages|heads"),
])
def test_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        _attend(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(k=lambda t: t.float()), "key"), (dict(v=lambda t: t.float()), "value"), (dict(v=lambda t: t[:2]), "value"), (dict(v=lambda t: t[:, :1]), "value"),
    (dict(k=lambda t: torch.zeros(5, KV, 96, dtype=BF16)), "value|head_dim"), (dict(gk=lambda t: t.to(BF16)), "gamma_k"), (dict(gk=lambda t: t[:32]), "gamma_k"),
    (dict(gq=lambda t: torch.ones(128)[::2]), "gamma_q"), (dict(freqs=lambda t: t.double()), "freqs_cis"), (dict(freqs=lambda t: t[:2]), "freqs_cis"),
    (dict(freqs=lambda t: torch.zeros(5, 1, 24)), "freqs_cis"), (dict(freqs=lambda t: torch.zeros(5, 1, 80)), "freqs_cis"), (dict(freqs=lambda t: torch.zeros(())), "freqs_cis"),
    (dict(out=lambda t: None), "go together"), (dict(q=lambda t: None, out=lambda t: None), "go together"), (dict(out=lambda t: t[:1]), "query_out"),
    (dict(w=lambda t: t.half()), "key_weights"), (dict(w=lambda t: t[1:]), "key_weights"), (dict(w=lambda t: t[:, :, :32]), "key_weights"),
])
def test_write_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        _write(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(lse=lambda t: t[:1]), "lse"), (dict(lse=lambda t: t.half()), "lse"), (dict(w=lambda t: t.half()), "key_weights"), (dict(w=lambda t: t[0]), "heads"),
    (dict(w=lambda t: t[:-1]), "key_weights"), (dict(w=lambda t: t.transpose(1, 2)), "heads|key_weights"),
])
def test_weights_refuse(change, text):
    with pytest.raises(ValueError, match=text):
        _sum(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(w=lambda t: t.double()), "key_weights"), (dict(w=lambda t: t[0]), "kv_heads"), (dict(keep=lambda t: t.long()), "keep_lens"), (dict(keep=lambda t: t[:1]), "keep_lens"),
    (dict(kept=lambda t: t.float()), "kept_lens"), (dict(kept=lambda t: torch.zeros(4, dtype=I32)[::2]), "kept_lens"), (dict(to=lambda t: t.long()), "kept_table"),
    (dict(to=lambda t: t[:1]), "kept_table"), (dict(to=lambda t: t[0]), "kept_table"), (dict(slots=lambda t: t[..., :64]), "kept_slots"),
    (dict(slots=lambda t: t.long()), "kept_slots"), (dict(dim=lambda n: 96), "head_dim"), (dict(dim=lambda n: 128), "kv_pages"),
])
def test_eviction_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        _evict(_args(**change))


def test_eviction_refuses_a_negative_window():
    with pytest.raises(ValueError, match="recent"):
        _evict(_args(), recent=-1)


# ---- the C entries: a status and a message before any launch (pointers are only compared with null and for alignment)
def _attend_c(q=P, stride=512, heads=8, kv=2, dim=64, scale=0.1, out=P, ws=P, nbytes=1 << 40, **b):
    b = {**BATCH_C, **b}
    return (q, stride, b["pages"], b["n_pages"], b["table"], b["max_pages"], b["cu"], b["lens"], b["n_seqs"], b["n_tokens"], heads, kv, dim, scale,
            out, None, ws, nbytes, None)


def _write_c(k=P, ks=128, v=P, vs=128, q=P, qs=512, heads=8, kv=2, dim=64, rope=64, freqs=P, out=P, **b):
    b = {**BATCH_C, **b}
    return (k, ks, v, vs, b["pages"], b["n_pages"], b["table"], b["max_pages"], b["cu"], b["lens"], b["n_seqs"], b["n_tokens"], kv, dim, P, freqs, rope,
            q, qs, heads, P, out, P, 1e-6, 0, None)


def _sum_c(q=P, stride=512, lse=P, heads=8, kv=2, dim=64, scale=0.1, w=P, **b):
    b = {**BATCH_C, **b}
    return (q, stride, lse, b["pages"], b["n_pages"], b["table"], b["max_pages"], b["cu"], b["lens"], b["n_seqs"], b["n_tokens"], heads, kv, dim, scale,
            1, w, None)


def _evict_c(w=P, kv=2, dim=64, recent=0, to=P, kept_pages=3, kept=P, slots=P, **b):
    b = {**BATCH_C, **b}
    return (b["pages"], w, b["n_pages"], b["table"], b["max_pages"], b["lens"], b["cu"], b["n_seqs"], kv, dim, recent, to, kept_pages, kept, slots, None)


ENTRIES = [("tl_flash_paged_gqa", _attend_c), ("tl_gqa_cache_write", _write_c), ("tl_gqa_cache_weights", _sum_c)]


@pytest.mark.parametrize("name,args", [*ENTRIES, ("tl_gqa_cache_evict", _evict_c)])
@pytest.mark.parametrize("change,code,text", [
    (dict(pages=None), 1, "null pointer"), (dict(table=None), 1, "null pointer"), (dict(cu=None), 1, "null pointer"), (dict(lens=None), 1, "null pointer"),
    (dict(pages=P + 8), 1, "16-byte aligned"), (dict(n_pages=0), 1, "n_pages"), (dict(n_pages=1 << 31), 1, "n_pages"), (dict(max_pages=0), 1, "max_pages"),
    (dict(n_seqs=-1), 1, "out of range"), (dict(n_seqs=1 << 24), 1, "out of range"), (dict(dim=96), 3, "head_dim"), (dict(dim=256), 3, "head_dim"),
    (dict(kv=0), 3, "kv_heads"), (dict(kv=129), 3, "kv_heads"),
])
def test_c_entries_refuse_a_batch(name, args, change, code, text):
    _refused(name, args(**change), code, text)


@pytest.mark.parametrize("name,args", ENTRIES)
@pytest.mark.parametrize("change,code,text", [
    (dict(heads=0), 3, "heads"), (dict(heads=130), 3, "heads"), (dict(heads=7), 3, "multiple"), (dict(n_tokens=-1), 1, "out of range"),
    (dict(n_tokens=1 << 26), 1, "out of range"), (dict(n_tokens=1 << 24), 3, "rows|room"),
])
def test_c_entries_refuse_heads_and_tokens(name, args, change, code, text):
    lib = _lib.load()
    assert getattr(lib, name)(*args(**change)) == code
    assert any(t in lib.tl_last_error().decode() for t in text.split("|"))


@pytest.mark.parametrize("name,args,change,code,text", [
    ("tl_flash_paged_gqa", _attend_c, dict(q=None), 1, "null pointer"), ("tl_flash_paged_gqa", _attend_c, dict(out=None), 1, "null pointer"),
    ("tl_flash_paged_gqa", _attend_c, dict(q=P + 8), 1, "aligned"), ("tl_flash_paged_gqa", _attend_c, dict(out=P + 2), 1, "aligned"),
    ("tl_flash_paged_gqa", _attend_c, dict(stride=516), 1, "multiple of 8"), ("tl_flash_paged_gqa", _attend_c, dict(stride=504), 1, "no less"),
    ("tl_flash_paged_gqa", _attend_c, dict(scale=0.0), 1, "softmax_scale"), ("tl_flash_paged_gqa", _attend_c, dict(scale=float("nan")), 1, "softmax_scale"),
    ("tl_flash_paged_gqa", _attend_c, dict(max_pages=9, ws=None), 1, "workspace"), ("tl_flash_paged_gqa", _attend_c, dict(max_pages=9, nbytes=4096), 1, "workspace"),
    ("tl_flash_paged_gqa", _attend_c, dict(max_pages=9, ws=P + 8), 1, "workspace"), ("tl_flash_paged_gqa", _attend_c, dict(n_seqs=(1 << 16) + 1), 3, "sequences"),
    ("tl_flash_paged_gqa", _attend_c, dict(max_pages=(1 << 20) + 1), 3, "pages"),
    ("tl_gqa_cache_write", _write_c, dict(k=None), 1, "null pointer"), ("tl_gqa_cache_write", _write_c, dict(v=P + 4), 1, "aligned"),
    ("tl_gqa_cache_write", _write_c, dict(ks=100), 1, "multiple of 8"), ("tl_gqa_cache_write", _write_c, dict(vs=120), 1, "no less"),
    ("tl_gqa_cache_write", _write_c, dict(qs=500), 1, "query"), ("tl_gqa_cache_write", _write_c, dict(out=None), 1, "query_out"),
    ("tl_gqa_cache_write", _write_c, dict(rope=24), 3, "rope_dim"), ("tl_gqa_cache_write", _write_c, dict(rope=80), 3, "rope_dim"),
    ("tl_gqa_cache_write", _write_c, dict(rope=0), 3, "rope_dim"), ("tl_gqa_cache_write", _write_c, dict(n_tokens=5, n_seqs=(1 << 23) - 1), 3, "room"),
    ("tl_gqa_cache_weights", _sum_c, dict(lse=None), 1, "null pointer"), ("tl_gqa_cache_weights", _sum_c, dict(w=None), 1, "null pointer"),
    ("tl_gqa_cache_weights", _sum_c, dict(q=None), 1, "null pointer"), ("tl_gqa_cache_weights", _sum_c, dict(scale=-1.0), 1, "softmax_scale"),
    ("tl_gqa_cache_weights", _sum_c, dict(n_seqs=(1 << 16) + 1), 3, "sequences"),
    ("tl_gqa_cache_evict", _evict_c, dict(w=None), 1, "null pointer"), ("tl_gqa_cache_evict", _evict_c, dict(to=None), 1, "null pointer"),
    ("tl_gqa_cache_evict", _evict_c, dict(kept=None), 1, "null pointer"), ("tl_gqa_cache_evict", _evict_c, dict(slots=None), 1, "null pointer"),
    ("tl_gqa_cache_evict", _evict_c, dict(recent=-1), 1, "recent"), ("tl_gqa_cache_evict", _evict_c, dict(recent=1 << 31), 1, "recent"),
    ("tl_gqa_cache_evict", _evict_c, dict(kept_pages=0), 1, "kept_pages"), ("tl_gqa_cache_evict", _evict_c, dict(kept_pages=1 << 25), 1, "kept_pages"),
    ("tl_gqa_cache_evict", _evict_c, dict(kept_pages=1 << 22), 3, "room"),
])
def test_c_entries_refuse(name, args, change, code, text):
    _refused(name, args(**change), code, text)


@pytest.mark.parametrize("name,args", ENTRIES)
@pytest.mark.parametrize("nothing", [dict(n_tokens=0), dict(n_seqs=0)])
def test_an_empty_batch_is_no_error(name, args, nothing):
    """Nothing is launched, and no pointer is asked for."""
    assert getattr(_lib.load(), name)(*args(**nothing, pages=None, table=None, cu=None, lens=None)) == 0


def test_no_sequence_to_evict_is_no_error():
    assert _lib.load().tl_gqa_cache_evict(*_evict_c(n_seqs=0, pages=None, table=None, cu=None, lens=None)) == 0


def test_the_workspace_follows_the_sizes():
    """None for short tables and for more sequences than a launch plans; for the others, no more than their pieces take."""
    f = _lib.load().tl_flash_paged_gqa_workspace_bytes
    assert f(1, 1, 8, 2, 64, 8) == 0 and f(1, 1, 8, 2, 64, 9) > 0
    assert f(512, 512, 8, 2, 64, 9) > 0 and f(513, 513, 8, 2, 64, 9) == 0
    assert f(1, 1, 8, 2, 64, 9) == f(1, 1, 8, 2, 64, 1 << 20) < f(1, 1, 8, 2, 128, 9)
    assert f(1, 1 << 20, 8, 2, 128, 1 << 20) < 1 << 27
    assert f(0, 1, 8, 2, 64, 9) == f(1, 0, 8, 2, 64, 9) == f(1, 1, 7, 2, 64, 9) == f(1, 1, 8, 2, 96, 9) == f(1, 1, 8, 0, 64, 9) == 0


def test_page_bytes():
    lib_sizes = [(1, 64), (1, 128), (2, 64), (8, 128), (16, 128), (17, 64), (128, 128)]
    for kv, dim in lib_sizes:
        assert gqa_page_bytes(kv, dim) == gqa.page_bytes(kv, dim) and gqa_page_bytes(kv, dim) % 128 == 0


def test_the_oracle_reads_what_the_page_layout_says():
    pages = torch.zeros(2, gqa.page_bytes(3, 64), dtype=torch.uint8)
    k, v, scales = gqa.views(pages, 3, 64)
    k[1, 2, 5, 7], v[1, 1, 7, 5], scales[1, 2, 1] = 0x38, 0x39, 1.0
    at = torch.nonzero(pages[1]).flatten().tolist()
    head, behind = 2 * 64 * 64, 3 * 2 * 64 * 64
    assert at == [head + 64 * 64 + 7 * 64 + 5, 2 * head + 5 * 64 + 7, behind + 2 * 8 + 4 + 2, behind + 2 * 8 + 4 + 3]
    assert not pages[0].any()


@pytest.mark.parametrize("amax,scale", [(0.0, 2.0 ** -22), (448.0, 1.0), (448.0 * (1 + 2 ** -20), 2.0), (449.0, 2.0), (1.75, 2.0 ** -8), (1.7500001, 2.0 ** -7),
                                        (3.3895e38, 2.0 ** 120), (1e-4, 2.0 ** -22)])
def test_the_least_scale(amax, scale):
    assert gqa.scale_of(amax) == scale and max(amax, 1e-4) <= 448 * scale


@pytest.mark.parametrize("off", [0, 4, -4])
def test_eviction_refuses_new_lengths_in_the_old_ones_place(off):
    """A head's workgroup may still read a length when another one's has written the new one."""
    _refused("tl_gqa_cache_evict", _evict_c(n_seqs=2, lens=P, kept=P + off), 1, "kept_lens")


@pytest.mark.parametrize("name,args", [("tl_flash_paged_gqa", _attend_c), ("tl_gqa_cache_weights", _sum_c)])
@pytest.mark.parametrize("scale", [2.4e38, 3.4e38, float("inf")])
def test_a_softmax_scale_that_passes_fp32_times_log2_e(name, args, scale):
    """The exponents are powers of two: an infinite factor would make the scores of zero queries NaN."""
    _refused(name, args(scale=scale), 1, "softmax_scale")


@pytest.mark.parametrize("off", [4, -4])
def test_eviction_refuses_new_lengths_that_overlap_the_counts_of_others(off):
    """The counts' own place is fine: a length in its sequence's count's place brings out itself.  One further, it is another's count."""
    _refused("tl_gqa_cache_evict", _evict_c(n_seqs=2, lens=P + 4096, cu=P, kept=P + off), 1, "kept_lens")
