"""Refusals of the paged-cache ops and the sampled pick that need no GPU: the C entries check
their arguments before any CUDA call, and the Python ops before any entry."""

from __future__ import annotations

import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]
P = ctypes.c_void_p(4096)  # a non-null address that no entry reads on the host


def _pages(**kw):
    from gpu.nf4._lib import ChrNf4Pages

    d = dict(k=4096, v=4096, table=4096, k_page_stride=16 * 2 * 64, v_page_stride=16 * 2 * 64, table_stride=4, n_pages=8,
             page=16, n_kv=2, hd=64, batch=2, max_pages=4)
    d.update(kw)
    return ChrNf4Pages(**d)


def _append(pages=None, **kw):
    from gpu.nf4 import _lib

    d = dict(q=4096, q_stride=512, k=4096, k_stride=128, v=4096, v_stride=128, q_out=4096, q_out_stride=512, cos=4096,
             sin=4096, tab_stride=32, tab_rows=64, tab_f32=1, rot=64, seq=4096, slot=4096, T=3, n_q=8)
    d.update(kw)
    args = _lib.ChrNf4RopeKvPaged(pages=_pages() if pages is None else pages, **d)
    return _lib.load().chr_nf4_rope_kv_paged(ctypes.byref(args), None)


def _attn(pages=None, **kw):
    from gpu.nf4 import _lib

    d = dict(q=4096, q_stride=512, out=4096, q_start=4096, kv_len=4096, T=3, n_q=8, scale=0.1, ws=4096, ws_floats=1 << 30)
    d.update(kw)
    args = _lib.ChrNf4AttnPaged(pages=_pages() if pages is None else pages, **d)
    return _lib.load().chr_nf4_attn_paged(ctypes.byref(args), None)


def _sample(**kw):
    from gpu.nf4 import _lib

    d = dict(logits=P, rs=100, n=100, batch=2, u=P, t=None, k=None, p=None, m=None, prob=None, nxt=P, tok=None, pos=None,
             fin=None, eos=-1)
    d.update(kw)
    return _lib.load().chr_nf4_sample_commit_batch(*d.values(), None)


@pytest.mark.parametrize("bad", [dict(page=8), dict(page=24), dict(page=1 << 17), dict(n_pages=0), dict(n_kv=0), dict(hd=63),
                                 dict(batch=0), dict(max_pages=0), dict(table_stride=3), dict(k_page_stride=100),
                                 dict(v_page_stride=2047), dict(max_pages=1 << 28, table_stride=1 << 28)])
def test_a_cache_that_is_none_is_refused(bad):
    assert _append(_pages(**bad)) == -3 and _attn(_pages(**bad)) == -3


@pytest.mark.parametrize("null", ["k", "v", "table"])
def test_null_pools_are_refused(null):
    assert _append(_pages(**{null: None})) == -1 and _attn(_pages(**{null: None})) == -1


@pytest.mark.parametrize("kw,rc", [(dict(k=None), -1), (dict(v=None), -1), (dict(q=None), -1), (dict(q_out=None), -1),
                                   (dict(cos=None), -1), (dict(sin=None), -1), (dict(slot=None), -1), (dict(T=0), -3),
                                   (dict(n_q=-1), -3), (dict(rot=0), -3), (dict(rot=3), -3), (dict(rot=66), -3),
                                   (dict(tab_stride=31), -3), (dict(tab_rows=0), -3), (dict(q_stride=511), -3),
                                   (dict(k_stride=127), -3), (dict(v_stride=127), -3), (dict(q_out_stride=511), -3),
                                   (dict(seq=None), -3)])
def test_append_refusals(kw, rc):
    assert _append(**kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(q=None), -1), (dict(out=None), -1), (dict(kv_len=None), -1), (dict(ws=None), -1),
                                   (dict(T=0), -3), (dict(n_q=0), -3), (dict(n_q=7), -3), (dict(q_stride=511), -3),
                                   (dict(tree=4096), -3), (dict(tree=4096, tree_words=(1 << 24) + 1), -3),
                                   (dict(scale=float("nan")), -3), (dict(scale=float("inf")), -3),
                                   (dict(q_start=None), -3), (dict(T=1 << 30), -3), (dict(q=4098), -5), (dict(out=4104), -5),
                                   (dict(q_stride=516), -5), (dict(ws=4104), -5), (dict(tree=4100, tree_words=1), -5),
                                   (dict(ws_floats=0), -7)])
def test_attention_refusals(kw, rc):
    assert _attn(**kw) == rc


@pytest.mark.parametrize("hd", [8, 24, 48, 96, 256])
def test_attention_refuses_other_head_dims(hd):
    assert _attn(_pages(hd=hd, k_page_stride=1 << 16, v_page_stride=1 << 16), q_stride=1 << 14) == -3


def test_attention_refuses_unaligned_pools():
    assert _attn(_pages(k=4098)) == -5 and _attn(_pages(v=4104)) == -5
    assert _attn(_pages(k_page_stride=16 * 2 * 64 + 4)) == -5


def test_workspace_query_answers_zero_for_what_the_call_refuses():
    from gpu.nf4 import _lib

    ws = _lib.load().chr_nf4_attn_paged_ws
    assert ws(3, 2, 8, 2, 64) > 0
    for bad in ((0, 2, 8, 2, 64), (3, 0, 8, 2, 64), (3, 2, 7, 2, 64), (3, 2, 8, 0, 64), (3, 2, 8, 2, 48)):
        assert ws(*bad) == 0


@pytest.mark.parametrize("kw,rc", [(dict(logits=None), -1), (dict(u=None), -1), (dict(nxt=None), -1), (dict(n=0), -3),
                                   (dict(n=524281, rs=524281), -3), (dict(batch=0), -3), (dict(batch=65536), -3),
                                   (dict(rs=99), -3)])
def test_sample_refusals(kw, rc):
    assert _sample(**kw) == rc


def test_python_ops_refuse_cpu_tensors():
    from gpu.nf4 import nf4_attn_paged, nf4_rope_kv_paged, nf4_sample_commit_batch

    pool = torch.zeros((4, 16, 2, 64), dtype=torch.bfloat16)
    table = torch.zeros((2, 2), dtype=torch.int32)
    rows = torch.zeros((2, 2, 64), dtype=torch.bfloat16)
    tab = torch.zeros((32, 32))
    with pytest.raises(RuntimeError, match="CUDA"):
        nf4_rope_kv_paged(rows, rows, rows, pool, pool, table, tab, tab, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="CUDA"):
        nf4_attn_paged(rows, pool, pool, table, torch.zeros(2, dtype=torch.int32), 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        nf4_sample_commit_batch(torch.zeros((2, 8), dtype=torch.bfloat16), torch.zeros(2), torch.zeros(2, dtype=torch.int64))


@pytest.mark.parametrize("mirror,name", [("ChrNf4Pages", "chr_nf4_pages_t"), ("ChrNf4RopeKvPaged", "chr_nf4_rope_kv_paged_t"),
                                         ("ChrNf4AttnPaged", "chr_nf4_attn_paged_t")])
def test_records_match_the_header(mirror, name, tmp_path):
    from gpu.nf4 import _lib

    cls = getattr(_lib, mirror)
    src = tmp_path / "sz.c"
    fields = [f[0] for f in cls._fields_]
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "chr_gpu.h"\nint main(void) { printf("%zu", '
                   f"sizeof({name}));\n"
                   + "".join(f'printf(" %zu", offsetof({name}, {f}));\n' for f in fields) + "return 0; }\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_records_are_packed_in_the_order_of_their_fields():
    from gpu.nf4 import _lib
    from gpu.nf4.paged import _ATTN, _ROPE

    def flat(record):
        for name, _ in record._fields_:
            v = getattr(record, name)
            yield from flat(v) if isinstance(v, ctypes.Structure) else [v]

    for pack, cls, n in ((_ROPE, _lib.ChrNf4RopeKvPaged, 34), (_ATTN, _lib.ChrNf4AttnPaged, 26)):
        values = list(range(1, n + 1))
        assert list(flat(cls.from_buffer_copy(pack(*values)))) == values


def test_overlap_of_row_views():
    from gpu.nf4.paged import _overlap

    flat = torch.empty(1000, dtype=torch.bfloat16)

    def both(a, b, row):
        args = [(t.data_ptr(), t.shape[0], t.stride(0)) for t in (a, b)]
        got = _overlap(*args[0], *args[1], row)
        assert got == _overlap(*args[1], *args[0], row)
        return got

    y = flat[:600].view(6, 100)
    q, k = y[:, :40], y[:, 60:]
    assert not both(q, k, 40)                       # side by side in one product
    assert both(q, y[3:, :40], 40) and both(q, q, 40)
    assert both(q, y[:, 30:70], 40)
    assert not both(y[:3], y[3:], 100)              # one behind the other
    assert both(flat[:240].view(4, 60), flat[:300].view(3, 100)[:, :60], 60)  # steps that differ
    assert not both(flat[:200].view(2, 100)[:, :60], flat[200:320].view(2, 60), 60)
