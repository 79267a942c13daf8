"""Ops of a paged KV cache and of the sampled pick, beside the dense-cache ops of this package.

Additive: the reference keeps one ``[max_seq, n_kv, hd]`` block per sequence
(gpu/decodev2/kv.py:14-120) and picks the argmax (gpu/decodev2/step.py:182). A cache is two
pools of pages ``[n_pages, page, n_kv, hd]`` and a table ``[batch, max_pages]`` of page ids;
cache row ``a`` of sequence ``s`` is row ``a % page`` of page ``table[s, a // page]``.

As everywhere in this package the ops check their arguments before anything is launched, run
on torch's current stream of the tensors' device, and have no fallback. What lies on the
device (ids, slots, lengths, tables, masks) is read there at launch, so that a captured graph
follows what the tensors hold at replay.
"""

from __future__ import annotations

import functools

import torch

from . import _lib
from ._lib import ChrNf4Pages

__all__ = ["nf4_attn_paged", "nf4_rope_kv_paged", "nf4_sample_commit_batch", "PAGED_HEAD_DIMS", "SAMPLE_MAX_VOCAB"]

#: head dims the attention covers
PAGED_HEAD_DIMS = (16, 32, 64, 128)
#: widest row the sampled pick takes
SAMPLE_MAX_VOCAB = 524280

_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


def _fail(msg: str):
    raise RuntimeError(msg)


# The host's share of a small call is longer than the kernel's: the raw forms of "current device"
# and "current stream" take a tenth of what the public ones do.
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, device: torch.device, *args) -> None:
    """``name(*args, stream)`` with ``device`` current, on its current stream."""
    index = device.index
    fn = getattr(_lib.load(), name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc, name)


def _on(t: torch.Tensor, device: torch.device, dtype: torch.dtype, what: str) -> None:
    if t.dtype is not dtype or t.device != device:
        _fail(f"{what} must be {str(dtype)[6:]} on {device}")


def _vector(t: torch.Tensor | None, n: int, device: torch.device, dtype: torch.dtype, what: str) -> int:
    """Address of a contiguous vector of ``n`` elements; 0 for ``None``."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.device != device or t.numel() != n or not t.is_contiguous():
        _fail(f"{what} must be contiguous {str(dtype)[6:]} of {n} elements on {device}")
    return t.data_ptr()


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor) -> tuple[ChrNf4Pages, torch.device]:
    if not k_pages.is_cuda or k_pages.dtype is not _BF16 or k_pages.dim() != 4:
        _fail("k_pages must be a CUDA bfloat16 [n_pages, page, n_kv, hd]")
    device = k_pages.device
    shape = k_pages.shape
    n_pages, page, n_kv, hd = shape
    _on(v_pages, device, _BF16, "v_pages")
    if v_pages.shape != shape:
        _fail("k_pages and v_pages differ in shape")
    inner = (n_kv * hd, hd, 1)
    ks, vs = k_pages.stride(), v_pages.stride()
    if ks[1:] != inner or vs[1:] != inner:
        _fail("the pages of a pool must each be contiguous")
    if page < 16 or page & (page - 1) or page > 65536:
        _fail(f"page must be a power of two in 16..65536, got {page}")
    _on(table, device, _I32, "page_table")
    if table.dim() != 2 or table.stride(1) != 1:
        _fail("page_table must be int32 [batch, max_pages] with contiguous rows")
    batch, max_pages = table.shape
    if n_pages < 1 or batch < 1 or max_pages < 1:
        _fail("the pools and page_table must not be empty")
    one = page * n_kv * hd
    t_stride = table.stride(0)
    if (n_pages > 1 and (ks[0] < one or vs[0] < one)) or (batch > 1 and t_stride < max_pages):
        _fail("pages or table rows overlap")
    return ChrNf4Pages(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), max(ks[0], one), max(vs[0], one),
                       max(t_stride, max_pages), n_pages, page, n_kv, hd, batch, max_pages), device


def _head_rows(t: torch.Tensor, hd: int, device: torch.device, what: str) -> tuple[int, int, int]:
    """(rows, heads, row stride) of a bf16 ``[T, heads, hd]`` or ``[T, heads*hd]`` view whose rows
    are contiguous."""
    _on(t, device, _BF16, what)
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        rows, heads, width = shape
        if width != hd or stride[2] != 1 or (heads > 1 and stride[1] != hd):
            _fail(f"{what} must be [T, heads, {hd}] with contiguous rows")
        row = heads * hd
    elif len(shape) == 2:
        rows, row = shape
        if row % hd or stride[1] != 1:
            _fail(f"{what} must be [T, heads*{hd}] with contiguous rows")
        heads = row // hd
    else:
        _fail(f"{what} must be [T, heads, hd] or [T, heads*hd]")
    if rows > 1 and stride[0] < row:
        _fail(f"{what} rows overlap")
    return rows, heads, max(stride[0], row)


def nf4_rope_kv_paged(
    q: torch.Tensor | None,
    k: torch.Tensor,
    v: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    slot: torch.Tensor,
    *,
    seq: torch.Tensor | None = None,
    position: torch.Tensor | None = None,
    interleaved: bool = False,
    q_out: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Rotary positions for ``T`` rows and the append of their k and v to a paged cache.

    Row ``t`` of ``q`` ``[T, n_q, hd]`` (or ``None``), ``k`` and ``v`` ``[T, n_kv, hd]`` (row views
    of a stacked product will do) belongs to sequence ``seq[t]`` (int32; default ``t``), takes its
    cache row ``slot[t]`` (int64) and is rotated for ``position[t]`` (int64; default ``slot[t]``).
    ``cos`` / ``sin`` ``[positions, rot/2]``, float32 or bfloat16 (``rope_tables_scaled``, or the
    first ``hd/2`` columns of the dense path's tables), rotate the first ``rot`` elements of every
    head: element ``i`` with ``i + rot/2``, or ``2i`` with ``2i + 1`` when ``interleaved``.
    Products and sum are float32, rounded once. Returns the rotated q ``[T, n_q, hd]``:
    ``q_out`` when given (may be ``q``), else a new tensor.

    A row whose sequence, slot, position or page lies outside (``seq`` -1 marks padding) is
    skipped: no cache row is written, its row of a given ``q_out`` is left alone, of a new one
    zero. Rows of one call must take different cache rows. See ``chr_nf4_rope_kv_paged``."""
    pages, device = _pages(k_pages, v_pages, page_table)
    hd = pages.hd
    rows, heads, ks = _head_rows(k, hd, device, "k")
    v_rows, v_heads, vs = _head_rows(v, hd, device, "v")
    if heads != pages.n_kv or v_heads != heads or v_rows != rows:
        _fail("k and v must have the pools' n_kv heads and the same rows")
    if rows < 1:
        _fail("k must have rows")
    if seq is None and rows > pages.batch:
        _fail(f"{rows} rows for {pages.batch} sequences need seq")
    if cos.dim() != 2 or cos.shape != sin.shape or cos.stride() != sin.stride() or cos.stride(1) != 1:
        _fail("cos and sin must be [positions, rot/2] of one layout with contiguous rows")
    if cos.dtype is not _F32 and cos.dtype is not _BF16:
        _fail("cos and sin must be float32 or bfloat16")
    _on(cos, device, cos.dtype, "cos")
    _on(sin, device, cos.dtype, "sin")
    tab_rows, half = cos.shape
    tab_stride = cos.stride(0)
    if tab_rows < 1 or half < 1 or 2 * half > hd or (tab_rows > 1 and tab_stride < half):
        _fail(f"cos and sin must have 1..{hd // 2} columns and positions")
    n_q = qs = os_ = 0
    zero = 0
    if q is not None:
        q_rows, n_q, qs = _head_rows(q, hd, device, "q")
        if q_rows != rows or n_q < 1:
            _fail("q must have k's rows")
        if q_out is None:
            q_out = torch.empty((rows, n_q, hd), dtype=_BF16, device=device)
            os_, zero = n_q * hd, 1
        else:
            o_rows, o_heads, os_ = _head_rows(q_out, hd, device, "q_out")
            if o_rows != rows or o_heads != n_q:
                _fail("q_out must have q's shape")
    elif q_out is not None:
        _fail("q_out goes with q")
    _call("chr_nf4_rope_kv_paged", device, pages, 0 if q is None else q.data_ptr(), qs, k.data_ptr(), ks,
          v.data_ptr(), vs, 0 if q is None else q_out.data_ptr(), os_, cos.data_ptr(), sin.data_ptr(),
          max(tab_stride, half), tab_rows, 1 if cos.dtype is _F32 else 0, 2 * half, 1 if interleaved else 0,
          _vector(seq, rows, device, _I32, "seq"), _vector(slot, rows, device, _I64, "slot"),
          _vector(position, rows, device, _I64, "position"), rows, n_q, zero)
    return q_out


def nf4_attn_paged(
    q: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    page_table: torch.Tensor,
    kv_len: torch.Tensor,
    scale: float,
    *,
    q_start: torch.Tensor | None = None,
    tree: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """GQA attention of the new rows of a batch of sequences over a paged cache -> ``[T, n_q*hd]``.

    Sequence ``b`` owns the rows ``q_start[b]:q_start[b+1]`` of ``q`` ``[T, n_q, hd]`` (int32
    ``[batch+1]``; default: one row each) and ``kv_len[b]`` cache rows (int32 ``[batch]``), the new
    rows' own being the last of them. Every new row sees the older cache rows and, of the new
    ones, itself and those before it; or, with ``tree`` (int64 ``[T, words]``), those whose bit is
    set in its mask: bit ``j % 64`` of word ``j // 64`` stands for the sequence's ``j``-th new row.
    One token per sequence is a decode step, a tree of drafted tokens is checked in one pass,
    and without ``tree`` many rows are a prompt chunk.

    A row that sees nothing gives zeros. Rows of ``q`` behind the last sequence's are left alone in
    a given ``out`` (which must not overlap ``q``), zero in a new one. See ``chr_nf4_attn_paged``."""
    pages, device = _pages(k_pages, v_pages, page_table)
    hd, batch = pages.hd, pages.batch
    if hd not in PAGED_HEAD_DIMS:
        _fail(f"head_dim must be one of {PAGED_HEAD_DIMS}, got {hd}")
    rows, n_q, qs = _head_rows(q, hd, device, "q")
    if rows < 1 or n_q < 1 or n_q % pages.n_kv:
        _fail("q must have rows and a multiple of the pools' n_kv heads")
    words = 0
    if tree is not None:
        if tree.dtype is not _I64 or tree.device != device or tree.dim() != 2 or tree.size(0) != rows \
                or tree.size(1) < 1 or not tree.is_contiguous():
            _fail(f"tree must be contiguous int64 [{rows}, words] on {device}")
        words = tree.size(1)
    if q_start is None and rows != batch:
        _fail(f"{rows} rows for {batch} sequences need q_start")
    zero = 0
    if out is None:
        out = torch.empty((rows, n_q * hd), dtype=_BF16, device=device)
        zero = 1
    elif out.dtype is not _BF16 or out.device != device or out.numel() != rows * n_q * hd or not out.is_contiguous():
        _fail(f"out must be contiguous bfloat16 [{rows}, {n_q * hd}] on {device}")
    need = _ws_floats(device.index, rows, batch, n_q, pages.n_kv, hd, pages.max_pages * pages.page)
    ws = torch.empty(need, dtype=_F32, device=device)
    _call("chr_nf4_attn_paged", device, pages, q.data_ptr(), qs, out.data_ptr(),
          _vector(q_start, batch + 1, device, _I32, "q_start"), _vector(kv_len, batch, device, _I32, "kv_len"),
          0 if tree is None else tree.data_ptr(), words, rows, n_q, float(scale), ws.data_ptr(), need, zero)
    return out


@functools.lru_cache(maxsize=4096)
def _ws_floats(index: int, rows: int, batch: int, n_q: int, n_kv: int, hd: int, cap: int) -> int:
    with torch.cuda.device(index):
        return int(_lib.load().chr_nf4_attn_paged_ws(rows, batch, n_q, n_kv, hd, cap))


def nf4_sample_commit_batch(
    logits: torch.Tensor,
    u: torch.Tensor,
    next_token: torch.Tensor,
    *,
    temperature: torch.Tensor | None = None,
    top_k: torch.Tensor | None = None,
    top_p: torch.Tensor | None = None,
    min_p: torch.Tensor | None = None,
    prob: torch.Tensor | None = None,
    token: torch.Tensor | None = None,
    position: torch.Tensor | None = None,
    finished: torch.Tensor | None = None,
    eos: int = -1,
) -> None:
    """Draws ``next_token`` (int64 ``[B]``) for every row of ``logits`` (bf16 ``[B, n]``, rows may
    be strided) with the row's own settings and its own uniform number ``u`` (float32 ``[B]`` in
    ``[0, 1)``), then commits it as :func:`nf4_pick_commit_batch` does.

    Tokens are ordered by logit (highest first, lowest index on ties); ``top_k`` (int32, 0: off),
    ``top_p`` (float32, 1: off) and ``min_p`` (float32 against the likeliest token, 0: off) each
    keep a beginning of that order, and the draw inverts its cumulative distribution at ``u``.
    A ``temperature`` (float32; default 1) of 0 picks greedily. ``prob`` (float32 ``[B]``) receives
    the probability the token was drawn with. The same inputs give the same tokens. See
    ``chr_nf4_sample_commit_batch``."""
    if not logits.is_cuda or logits.dtype is not _BF16 or logits.dim() != 2 or logits.stride(1) != 1:
        _fail("logits must be a CUDA bfloat16 [B, n] view with contiguous rows")
    b, n = logits.shape
    if b < 1 or not 1 <= n <= SAMPLE_MAX_VOCAB:
        _fail(f"logits must have rows of 1..{SAMPLE_MAX_VOCAB} tokens")
    device, stride = logits.device, logits.stride(0)
    if b > 1 and stride < n:
        _fail("logits rows overlap")
    if u is None or next_token is None:
        _fail("u and next_token are needed")
    _call("chr_nf4_sample_commit_batch", device, logits.data_ptr(), max(stride, n), n, b,
          _vector(u, b, device, _F32, "u"), _vector(temperature, b, device, _F32, "temperature"),
          _vector(top_k, b, device, _I32, "top_k"), _vector(top_p, b, device, _F32, "top_p"),
          _vector(min_p, b, device, _F32, "min_p"), _vector(prob, b, device, _F32, "prob"),
          _vector(next_token, b, device, _I64, "next_token"), _vector(token, b, device, _I64, "token"),
          _vector(position, b, device, _I64, "position"), _vector(finished, b, device, _U8, "finished"), int(eos))
