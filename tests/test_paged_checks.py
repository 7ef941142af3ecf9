"""Refusals of the paged latent cache's operators and of add_rmsnorm_quant: the wrappers' and the C entries' argument
checks, which need no GPU, and the device that a launch goes to."""
import contextlib

import pytest
import torch

from oracle import paged
from tests import _paged
from tilert_amd import _lib, kernel
from tilert_amd.flash_paged_mla import flash_paged_mla
from tilert_amd.mla_cache import mla_cache_read, mla_cache_write
from tilert_amd.rmsnorm import add_rmsnorm_quant

BF16, F32, I32, FP8 = torch.bfloat16, torch.float32, torch.int32, torch.float8_e4m3fn


def _args(**changes):
    """Arguments that pass every check but that of the device."""
    pages, table, cu, lens, rows = _paged.batch([2, 3], [70, 3])
    a = dict(q=torch.zeros(rows, 16, 512, dtype=BF16), qp=torch.zeros(rows, 16, 64, dtype=BF16), pages=pages, table=table,
             cu=cu, lens=lens, out=torch.zeros(rows, 16, 512, dtype=BF16), lse=torch.zeros(rows, 16),
             kv=torch.zeros(rows, 512, dtype=BF16), pe=torch.zeros(rows, 64, dtype=BF16), gamma=torch.ones(512),
             freqs=torch.zeros(rows, 1, 64))
    for k, f in changes.items():
        a[k] = f(a[k])
    return a


def _attend(a, **kw):
    flash_paged_mla(a["q"], a["qp"], a["pages"], a["table"], a["cu"], a["lens"], a["out"], a["lse"],
                    **{"model_arch": "deepseek_v3_2", **kw})


def _write(a, **kw):
    mla_cache_write(a["kv"], a["pe"], a["pages"], a["table"], a["cu"], a["lens"], a["gamma"], a["freqs"], **kw)


def _read(a):
    mla_cache_read(a["pages"], a["table"], a["cu"], a["lens"], a["kv"], a["pe"])


BATCH = [
    (dict(pages=lambda t: t.to(torch.int8)), "contiguous uint8"), (dict(pages=lambda t: t[:, :-16]), "contiguous uint8"),
    (dict(pages=lambda t: t[::2]), "contiguous uint8"), (dict(pages=lambda t: t.flatten()), "contiguous uint8"),
    (dict(table=lambda t: t.long()), "int32"), (dict(cu=lambda t: t.long()), "int32"), (dict(lens=lambda t: t.float()), "int32"),
    (dict(table=lambda t: t.T), "contiguous"), (dict(table=lambda t: t[0]), "sequences, max_pages"),
    (dict(cu=lambda t: t[:-1]), "cu_seqlens"), (dict(cu=lambda t: torch.cat([t, t])[::2]), "contiguous"),
    (dict(lens=lambda t: t[:1]), "seq_lens"), (dict(table=lambda t: t[:1]), "cu_seqlens"),
]


@pytest.mark.parametrize("change,text", BATCH)
@pytest.mark.parametrize("op", [_attend, _write, _read])
def test_a_batch_that_is_not_one(op, change, text):
    with pytest.raises(ValueError, match=text):
        op(_args(**change))


@pytest.mark.parametrize("op", [_attend, _write, _read])
def test_tensors_off_the_gpu(op):
    with pytest.raises(ValueError, match="GPU"):
        op(_args())


@pytest.mark.parametrize("change,text", [
    (dict(q=lambda t: t.half()), "bfloat16"), (dict(qp=lambda t: t.float()), "bfloat16"), (dict(out=lambda t: t.float()), "bfloat16"),
    (dict(q=lambda t: t[..., :256]), "512-wide"), (dict(qp=lambda t: t[..., :32]), "64-wide"),
    (dict(q=lambda t: t.transpose(0, 1)), "contiguous"), (dict(qp=lambda t: t[:, ::2]), "contiguous"),
    (dict(out=lambda t: t.transpose(0, 1)), "contiguous"), (dict(qp=lambda t: t[:1]), "tokens and heads"),
    (dict(out=lambda t: t[:1]), "query's shape"), (dict(q=lambda t: torch.zeros(5, 0, 512, dtype=BF16)), "heads"),
    (dict(q=lambda t: torch.zeros(5, 129, 512, dtype=BF16)), "heads"), (dict(q=lambda t: t[0, 0]), "512-wide"),
    (dict(lse=lambda t: t[:1]), "lse"), (dict(lse=lambda t: t.double()), "lse"), (dict(lse=lambda t: torch.zeros(16, 5).T), "lse"),
])
def test_attention_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        _attend(_args(**change))


def test_attention_refuses_other_kernels_and_models():
    with pytest.raises(ValueError, match="compute_kernel_type"):
        _attend(_args(), compute_kernel_type="fp8mma")


@pytest.mark.parametrize("change,text", [
    (dict(kv=lambda t: t.float()), "bfloat16"), (dict(pe=lambda t: t.float()), "bfloat16"), (dict(kv=lambda t: t[:, :500]), "latent"),
    (dict(pe=lambda t: t[:, :32]), "rope"), (dict(kv=lambda t: t[::2]), "contiguous"), (dict(pe=lambda t: t[:2]), "as many"),
])
@pytest.mark.parametrize("op", [_write, _read])
def test_rows_that_do_not_fit(op, change, text):
    with pytest.raises(ValueError, match=text):
        op(_args(**change))


@pytest.mark.parametrize("change,text", [
    (dict(gamma=lambda t: t.to(BF16)), "gamma"), (dict(gamma=lambda t: t[:256]), "gamma"), (dict(gamma=lambda t: torch.ones(1024)[::2]), "gamma"),
    (dict(freqs=lambda t: t.double()), "freqs_cis"), (dict(freqs=lambda t: t[:2]), "freqs_cis"),
])
def test_write_refuses(change, text):
    with pytest.raises(ValueError, match=text):
        _write(_args(**change))


def _norm(rows=3, dim=256, logs=torch.zeros(1), **changes):
    a = dict(x=torch.zeros(rows, dim, dtype=BF16), r=torch.zeros(rows, dim, dtype=BF16), g=torch.ones(dim),
             s=torch.zeros(rows, dim, dtype=BF16), y=torch.zeros(rows, dim, dtype=BF16), q=torch.zeros(rows, dim, dtype=FP8),
             qs=torch.zeros(rows, dim // 128))
    for k, f in changes.items():
        a[k] = f(a[k])
    add_rmsnorm_quant(a["x"], a["r"], a["g"], a["s"], a["y"], a["q"], a["qs"], logs, model_arch="deepseek_v3_2")


@pytest.mark.parametrize("changes,text", [
    (dict(logs=None), "profile_logs"), (dict(x=lambda t: t.float()), "bfloat16"), (dict(r=lambda t: t[:2]), "one shape"),
    (dict(s=lambda t: t.half()), "bfloat16"), (dict(y=lambda t: t[:, :128]), "one shape"), (dict(g=lambda t: t[:128]), "gamma_in"),
    (dict(q=lambda t: None), "go together"), (dict(qs=lambda t: None), "go together"), (dict(q=lambda t: t.float()), "float8"),
    (dict(qs=lambda t: t.double()), "float32"), (dict(qs=lambda t: t[:1]), "dim // 128"), (dict(r=lambda t: t.T.contiguous().T), "contiguous"),
    (dict(y=lambda t: None, q=lambda t: None, qs=lambda t: None), "must be given"), (dict(), "GPU"),
])
def test_norm_refuses(changes, text):
    with pytest.raises(ValueError, match=text):
        _norm(**changes)


# ---- the C entries: a status and a message before any launch (pointers are only compared with null and for alignment)
P = 256


def _refused(name, args, code, text):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == code
    assert text in lib.tl_last_error().decode()


BATCH_C = dict(pages=P, n_pages=9, table=P, max_pages=3, cu=P, lens=P, n_seqs=2, n_tokens=5)


def _write_c(gamma=P, kv=P, pe=P, mode=2, **b):
    b = {**BATCH_C, **b}
    return (kv, pe, b["pages"], b["n_pages"], b["table"], b["max_pages"], b["cu"], b["lens"], b["n_seqs"], b["n_tokens"], gamma, P,
            1e-6, 1, mode, None)


def _read_c(kv=P, pe=P, **b):
    b = {**BATCH_C, **b}
    return (b["pages"], b["n_pages"], b["table"], b["max_pages"], b["cu"], b["lens"], b["n_seqs"], b["n_tokens"], kv, pe, None)


def _attend_c(q=P, qp=P, heads=16, scale=0.1, out=P, ws=P, nbytes=1 << 40, **b):
    b = {**BATCH_C, **b}
    return (q, qp, b["pages"], b["n_pages"], b["table"], b["max_pages"], b["cu"], b["lens"], b["n_seqs"], b["n_tokens"], heads, scale,
            out, None, ws, nbytes, None)


ENTRIES = [("tl_mla_cache_write", _write_c), ("tl_mla_cache_read", _read_c), ("tl_flash_paged_mla", _attend_c)]


@pytest.mark.parametrize("name,args", ENTRIES)
@pytest.mark.parametrize("change,text", [
    (dict(pages=None), "null pointer"), (dict(table=None), "null pointer"), (dict(cu=None), "null pointer"), (dict(lens=None), "null pointer"),
    (dict(pages=P + 8), "16-byte aligned"), (dict(n_pages=0), "n_pages"), (dict(n_pages=1 << 31), "n_pages"), (dict(max_pages=0), "max_pages"),
    (dict(max_pages=1 << 25), "max_pages"), (dict(n_seqs=-1), "out of range"), (dict(n_tokens=-1), "out of range"),
    (dict(n_seqs=1 << 24), "out of range"), (dict(n_tokens=1 << 31), "out of range"),
    (dict(n_tokens=1 << 26), "out of range"),
])
def test_c_entries_refuse_a_batch(name, args, change, text):
    _refused(name, args(**change), 1, text)


@pytest.mark.parametrize("name,args,change,code,text", [
    ("tl_mla_cache_write", _write_c, dict(kv=None), 1, "null pointer"), ("tl_mla_cache_write", _write_c, dict(pe=None), 1, "null pointer"),
    ("tl_mla_cache_write", _write_c, dict(kv=P + 2), 1, "aligned"), ("tl_mla_cache_write", _write_c, dict(gamma=P + 4), 1, "aligned"),
    ("tl_mla_cache_write", _write_c, dict(mode=3), 1, "scale_mode"), ("tl_mla_cache_write", _write_c, dict(mode=-1), 1, "scale_mode"),
    ("tl_mla_cache_read", _read_c, dict(kv=None), 1, "null pointer"), ("tl_mla_cache_read", _read_c, dict(pe=P + 8), 1, "aligned"),
    ("tl_flash_paged_mla", _attend_c, dict(heads=0), 3, "heads"), ("tl_flash_paged_mla", _attend_c, dict(heads=129), 3, "heads"),
    ("tl_flash_paged_mla", _attend_c, dict(q=None), 1, "null pointer"), ("tl_flash_paged_mla", _attend_c, dict(out=None), 1, "null pointer"),
    ("tl_flash_paged_mla", _attend_c, dict(q=P + 8), 1, "aligned"), ("tl_flash_paged_mla", _attend_c, dict(out=P + 8), 1, "aligned"),
    ("tl_flash_paged_mla", _attend_c, dict(scale=0.0), 1, "softmax_scale"), ("tl_flash_paged_mla", _attend_c, dict(scale=float("nan")), 1, "softmax_scale"),
    ("tl_flash_paged_mla", _attend_c, dict(scale=float("inf")), 1, "softmax_scale"), ("tl_flash_paged_mla", _attend_c, dict(max_pages=9, ws=None), 1, "workspace"),
    ("tl_flash_paged_mla", _attend_c, dict(max_pages=9, nbytes=4096), 1, "workspace"), ("tl_flash_paged_mla", _attend_c, dict(max_pages=9, ws=P + 8), 1, "aligned"),
    ("tl_flash_paged_mla", _attend_c, dict(n_tokens=1 << 24), 3, "rows"), ("tl_flash_paged_mla", _attend_c, dict(n_seqs=(1 << 20) + 1), 3, "sequences"),
    ("tl_flash_paged_mla", _attend_c, dict(max_pages=(1 << 20) + 1), 3, "pages"),
])
def test_c_entries_refuse(name, args, change, code, text):
    _refused(name, args(**change), code, text)


@pytest.mark.parametrize("name,args", ENTRIES)
@pytest.mark.parametrize("nothing", [dict(n_tokens=0), dict(n_seqs=0)])
def test_an_empty_batch_is_no_error(name, args, nothing):
    """Nothing is launched, and no pointer is asked for."""
    assert getattr(_lib.load(), name)(*args(**nothing, pages=None, table=None, cu=None, lens=None)) == 0


@pytest.mark.parametrize("change,text", [
    (dict(dim=100), "multiple of 128"), (dict(dim=0), "multiple of 128"), (dict(dim=16512), "at most"), (dict(rows=-1), "rows"), (dict(mode=3), "scale_mode"),
    (dict(x=None), "null pointer"), (dict(s=None), "null pointer"), (dict(y8=None), "null pointer"), (dict(ys=None), "null pointer"),
    (dict(y=None, y8=None, ys=None), "null pointer"), (dict(x=P + 8), "aligned"), (dict(y8=P + 8), "aligned"),
])
def test_c_norm_refuses(change, text):
    a = {**dict(x=P, r=P, g=P, rows=4, dim=256, s=P, y=P, y8=P, ys=P, mode=0), **change}
    _refused("tl_add_rmsnorm_quant", (a["x"], a["r"], a["g"], 1e-6, a["rows"], a["dim"], a["s"], a["y"], a["y8"], a["ys"], a["mode"], None), 1, text)


@pytest.mark.parametrize("rows,dim", [(1 << 24, 2048), (1 << 22, 2176), (1 << 22, 16384), (1 << 40, 128)])
def test_c_norm_refuses_more_rows_than_a_launch_has(rows, dim):
    _refused("tl_add_rmsnorm_quant", (P, P, P, 1e-6, rows, dim, P, P, P, P, 0, None), 3, "rows")


def test_the_workspace_follows_the_sizes():
    """None for short tables and for more row tiles than a split launch plans, one of a fixed size a tile height else."""
    f = _lib.load().tl_flash_paged_mla_workspace_bytes
    assert f(1, 1, 16, 8) == 0 and f(1, 1, 16, 9) > 0
    assert f(1, 1, 16, 9) == f(60, 60, 16, 4096) == f(1, 1, 16, 1 << 20)
    assert f(1, 8, 16, 9) == f(1, 2, 16, 9) < f(1, 9, 16, 9)
    assert f(1, 8188, 16, 512) > 0 and f(1, 8200, 16, 512) == 0 and f(2049, 2049, 16, 512) == 0
    assert f(0, 1, 16, 9) == f(1, 0, 16, 9) == f(1, 1, 0, 9) == f(1, 1, 129, 9) == 0


# ---- the device of a launch
class _OnDevice:
    def __init__(self, index):
        self.index = index

    def get_device(self):
        return self.index


def test_a_launch_goes_to_the_tensors_device(monkeypatch):
    current, seen = [0], []

    @contextlib.contextmanager
    def device(index):
        was, current[0] = current[0], index
        yield
        current[0] = was

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(_lib, "call", lambda name, *a: seen.append((name, a, current[0])))
    kernel._call(_OnDevice(0), "tl_x", 1)
    kernel._call(_OnDevice(1), "tl_y", 2)
    assert seen == [("tl_x", (1,), 0), ("tl_y", (2,), 1)] and current == [0]


def test_the_oracle_reads_what_the_page_layout_says():
    pages = torch.zeros(2, paged.PAGE_BYTES, dtype=torch.uint8)
    codes, scales, rope = paged.views(pages)
    codes.view(torch.uint8)[1, 2, 3], scales[1, 2], rope[1, 2, 3] = 0x38, 1.0, 1.0
    at = torch.nonzero(pages[1]).flatten().tolist()
    assert at == [2 * 512 + 3, 64 * 512 + 2 * 4 + 2, 64 * 512 + 2 * 4 + 3, 64 * 516 + (2 * 64 + 3) * 2, 64 * 516 + (2 * 64 + 3) * 2 + 1]
    assert not pages[0].any()
