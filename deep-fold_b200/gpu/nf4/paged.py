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
import struct

import torch

from . import _lib

__all__ = ["nf4_attn_paged", "nf4_attn_paged_status", "nf4_rope_kv_paged",
           "nf4_sample_commit_batch", "PAGED_HEAD_DIMS", "SAMPLE_MAX_VOCAB"]

#: head dims the attention covers
PAGED_HEAD_DIMS = (16, 32, 64, 128)
#: widest row the sampled pick takes
SAMPLE_MAX_VOCAB = 524280

_MOST = 0x7FFFFFFF  # counts are passed in 32 bits

_BF16, _F32, _I32, _I64, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.uint8


def _fail(msg: str):
    raise RuntimeError(msg)


# A small call takes longer on the host than on the device, so the host side is kept lean: device
# indices instead of device objects, each attribute read once, the raw forms of "current device"
# and "current stream", which take a tenth of what the public ones do, and the arguments packed into
# one record (ctypes takes 0.2 us to convert each argument of a call).
_PAGES = "6q6i"  # ChrNf4Pages
_ROPE = struct.Struct(_PAGES + "14q8i").pack  # ChrNf4RopeKvPaged
_ATTN = struct.Struct(_PAGES + "8q4ifi").pack  # ChrNf4AttnPaged
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


@functools.cache
def _entry(name: str):
    return getattr(_lib.load(), name)


def _call(name: str, index: int, *args) -> None:
    """``name(*args, stream)`` with device ``index`` current, on its current stream."""
    fn = _entry(name)
    if index == _current_device():
        rc = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    if rc != 0:
        _lib.check(rc, name)


def _vector(t: torch.Tensor | None, n: int, index: int, dtype: torch.dtype, what: str) -> int:
    """Address of a contiguous vector of ``n`` elements; 0 for ``None``."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != index or t.numel() != n or not t.is_contiguous():
        _fail(f"{what} must be contiguous {str(dtype)[6:]} of {n} elements on cuda:{index}")
    return t.data_ptr()


def _pages(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor) -> tuple[tuple, int]:
    """The fields of ``ChrNf4Pages`` for a paged cache, and its device's index."""
    index = k_pages.get_device()
    shape = k_pages.shape
    if index < 0 or k_pages.dtype is not _BF16 or len(shape) != 4:
        _fail("k_pages must be a CUDA bfloat16 [n_pages, page, n_kv, hd]")
    if v_pages.dtype is not _BF16 or v_pages.get_device() != index or v_pages.shape != shape:
        _fail(f"v_pages must be bfloat16 {list(shape)} on cuda:{index}, as k_pages")
    n_pages, page, n_kv, hd = shape
    one = page * n_kv * hd
    ks, k_row, k_head, k_el = k_pages.stride()
    vs, v_row, v_head, v_el = v_pages.stride()
    row = n_kv * hd
    if k_row != row or v_row != row or k_head != hd or v_head != hd or k_el != 1 or v_el != 1:
        _fail("the pages of a pool must each be contiguous")
    if page < 16 or page & (page - 1) or page > 65536:
        _fail(f"page must be a power of two in 16..65536, got {page}")
    if table.dtype is not _I32 or table.get_device() != index or table.dim() != 2:
        _fail(f"page_table must be int32 [batch, max_pages] on cuda:{index}")
    batch, max_pages = table.shape
    t_row, t_el = table.stride()
    if n_pages < 1 or batch < 1 or max_pages < 1 or one < 1:
        _fail("the pools and page_table must not be empty")
    if batch > _MOST or max_pages * page > _MOST:
        _fail("page_table is too large")
    if t_el != 1 and max_pages > 1:
        _fail("page_table must have contiguous rows")
    if ks < one or vs < one or t_row < max_pages:  # strides of an axis of one mean nothing
        if (n_pages > 1 and (ks < one or vs < one)) or (batch > 1 and t_row < max_pages):
            _fail("pages or table rows overlap")
        ks, vs, t_row = max(ks, one), max(vs, one), max(t_row, max_pages)
    return (k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), ks, vs, t_row, n_pages, page, n_kv, hd, batch,
            max_pages), index


def _head_rows(t: torch.Tensor, hd: int, index: int, what: str) -> tuple[int, int, int]:
    """(rows, heads, row stride) of a bf16 ``[T, heads, hd]`` or ``[T, heads*hd]`` view whose rows
    are contiguous."""
    shape, stride = t.shape, t.stride()
    if t.dtype is not _BF16 or t.get_device() != index:
        _fail(f"{what} must be bfloat16 on cuda:{index}")
    if len(shape) == 2:
        rows, row = shape
        heads, left = divmod(row, hd)
        if left or (stride[1] != 1 and row > 1):
            _fail(f"{what} must be [T, heads*{hd}] with contiguous rows")
    elif len(shape) == 3:
        rows, heads, width = shape
        row = heads * hd
        if width != hd or stride[2] != 1 or (stride[1] != hd and heads > 1):
            _fail(f"{what} must be [T, heads, {hd}] with contiguous rows")
    else:
        _fail(f"{what} must be [T, heads, hd] or [T, heads*hd]")
    step = stride[0]
    if rows > _MOST:
        _fail(f"{what} has too many rows")
    if step < row:
        if rows > 1:
            _fail(f"{what} rows overlap")
        step = row
    return rows, heads, step


def _overlap(a: int, a_rows: int, a_step: int, b: int, b_rows: int, b_step: int, row: int, b_row: int = 0) -> bool:
    """Whether two views of rows of ``row`` (``b``: ``b_row``, if given) bf16 elements, ``*_step`` apart, at
    addresses ``a`` and ``b`` share memory; views of one stacked product (one step, side by side) do not."""
    gap, b_row = (b - a) // 2, b_row or row
    if gap >= (a_rows - 1) * a_step + row or -gap >= (b_rows - 1) * b_step + b_row:
        return False
    if a_step == b_step:
        off = gap % a_step
        return off < row or off + b_row > a_step
    return True


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
    zero. Rows of one call must take different cache rows. ``q_out`` must not overlap ``k`` or ``v``,
    nor the pools each other; ``q``, ``k`` and ``v`` must not lie in cache rows the call writes. See
    ``chr_nf4_rope_kv_paged``."""
    pages, device = _pages(k_pages, v_pages, page_table)
    kp, vp, _, kps, vps, _, n_pages, page, n_kv, hd, batch, _ = pages
    rows, heads, ks = _head_rows(k, hd, device, "k")
    v_rows, v_heads, vs = _head_rows(v, hd, device, "v")
    if heads != n_kv or v_heads != heads or v_rows != rows:
        _fail("k and v must have the pools' n_kv heads and the same rows")
    if rows < 1:
        _fail("k must have rows")
    if seq is None and rows > batch:
        _fail(f"{rows} rows for {batch} sequences need seq")
    k_at, v_at = k.data_ptr(), v.data_ptr()
    gap = vp - kp
    if gap < 2 * kps * n_pages and -gap < 2 * vps * n_pages \
            and _overlap(kp, n_pages, kps, vp, n_pages, vps, page * n_kv * hd):
        _fail("k_pages and v_pages must not overlap")
    f32 = cos.dtype is _F32
    tab = cos.shape
    step = cos.stride()
    if (not f32 and cos.dtype is not _BF16) or sin.dtype is not cos.dtype or cos.get_device() != device \
            or sin.get_device() != device:
        _fail(f"cos and sin must be float32 or bfloat16, both on cuda:{device}")
    if len(tab) != 2 or sin.shape != tab or sin.stride() != step or (step[1] != 1 and tab[1] > 1):
        _fail("cos and sin must be [positions, rot/2] of one layout with contiguous rows")
    tab_rows, half = tab
    tab_stride = step[0]
    if not 1 <= tab_rows <= _MOST or half < 1 or 2 * half > hd or (tab_rows > 1 and tab_stride < half):
        _fail(f"cos and sin must have 1..{hd // 2} columns and positions")
    n_q = qs = os_ = zero = q_at = out_at = 0
    if q is not None:
        q_rows, n_q, qs = _head_rows(q, hd, device, "q")
        q_at = q.data_ptr()
        if q_rows != rows or n_q < 1:
            _fail("q must have k's rows")
        if q_out is None:
            q_out = q.new_empty((rows, n_q, hd))
            os_, zero, out_at = n_q * hd, 1, q_out.data_ptr()
        else:
            o_rows, o_heads, os_ = _head_rows(q_out, hd, device, "q_out")
            if o_rows != rows or o_heads != n_q:
                _fail("q_out must have q's shape")
            out_at = q_out.data_ptr()
            if (out_at != q_at or (os_ != qs and rows > 1)) and _overlap(out_at, rows, os_, q_at, rows, qs, n_q * hd):
                _fail("q_out must be q or not overlap it")
            # other threads read k and v in the same launch
            far = 2 * os_ * rows
            gap = k_at - out_at
            if gap < far and -gap < 2 * ks * rows and _overlap(out_at, rows, os_, k_at, rows, ks, n_q * hd, n_kv * hd):
                _fail("q_out must not overlap k")
            gap = v_at - out_at
            if gap < far and -gap < 2 * vs * rows and _overlap(out_at, rows, os_, v_at, rows, vs, n_q * hd, n_kv * hd):
                _fail("q_out must not overlap v")
    elif q_out is not None:
        _fail("q_out goes with q")
    _call("chr_nf4_rope_kv_paged", device, _ROPE(
        *pages, q_at, qs, k_at, ks, v_at, vs, out_at, os_, cos.data_ptr(), sin.data_ptr(),
        max(tab_stride, half), _vector(seq, rows, device, _I32, "seq"), _vector(slot, rows, device, _I64, "slot"),
        _vector(position, rows, device, _I64, "position"), tab_rows, f32, 2 * half, bool(interleaved), rows, n_q,
        zero, 0))
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

    Probabilities are rounded to bf16 for the value product, as the prompt attention of the dense
    cache does (its decode attention keeps them, and the query it rotates, in two bf16 terms). One form
    is chosen for the whole call from the mean rows per sequence: a long chunk and many single
    tokens go faster as two calls. A wait that runs out is reported by ``nf4_attn_paged_status``.

    A row that sees nothing gives zeros. Rows of ``q`` that no sequence owns (in front of
    ``q_start[0]``, from ``q_start[batch]`` on) are left alone in a given ``out`` (which must not
    overlap ``q``), zero in a new one. See ``chr_nf4_attn_paged``."""
    pages, device = _pages(k_pages, v_pages, page_table)
    n_kv, hd, batch = pages[8:11]
    if hd not in PAGED_HEAD_DIMS:
        _fail(f"head_dim must be one of {PAGED_HEAD_DIMS}, got {hd}")
    rows, n_q, qs = _head_rows(q, hd, device, "q")
    if rows < 1 or n_q < 1 or n_q % n_kv:
        _fail("q must have rows and a multiple of the pools' n_kv heads")
    words = 0
    if tree is not None:
        if tree.dtype is not _I64 or tree.get_device() != device or tree.dim() != 2 or tree.size(0) != rows \
                or tree.size(1) < 1 or not tree.is_contiguous():
            _fail(f"tree must be contiguous int64 [{rows}, words] on cuda:{device}")
        words = tree.size(1)
    if q_start is None and rows != batch:
        _fail(f"{rows} rows for {batch} sequences need q_start")
    zero = 0
    if out is None:
        out = q.new_empty((rows, n_q * hd))
        zero = 1
    elif out.dtype is not _BF16 or out.get_device() != device or out.numel() != rows * n_q * hd \
            or not out.is_contiguous():
        _fail(f"out must be contiguous bfloat16 [{rows}, {n_q * hd}] on cuda:{device}")
    elif _overlap(out.data_ptr(), rows, n_q * hd, q.data_ptr(), rows, qs, n_q * hd):
        _fail("out must not overlap q")
    scale = float(scale)
    if not -3e38 < scale < 3e38:
        _fail(f"scale must be finite, got {scale}")
    need = _ws_floats(device, rows, batch, n_q, n_kv, hd)
    ws = q.new_empty(need, dtype=_F32)
    _call("chr_nf4_attn_paged", device, _ATTN(
        *pages, q.data_ptr(), qs, out.data_ptr(), _vector(q_start, batch + 1, device, _I32, "q_start"),
        _vector(kv_len, batch, device, _I32, "kv_len"), 0 if tree is None else tree.data_ptr(), ws.data_ptr(), need,
        words, rows, n_q, zero, scale, 0))
    return out


@functools.lru_cache(maxsize=4096)
def _ws_floats(index: int, rows: int, batch: int, n_q: int, n_kv: int, hd: int) -> int:
    with torch.cuda.device(index):
        return int(_lib.load().chr_nf4_attn_paged_ws(rows, batch, n_q, n_kv, hd))


def nf4_attn_paged_status(device: torch.device | int | str | None = None) -> int:
    """Read and clear the paged attention's status word on ``device`` (default: the current one):
    0 = healthy, else a bounded wait of some launch since the last look ran out and that launch's
    output is undefined. Synchronises the device."""
    with torch.cuda.device(device):
        return int(_lib.load().chr_nf4_attn_paged_status())


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
    device = logits.get_device()
    if device < 0 or logits.dtype is not _BF16 or logits.dim() != 2:
        _fail("logits must be a CUDA bfloat16 [B, n]")
    b, n = logits.shape
    stride, el = logits.stride()
    if not 1 <= b <= 65535 or not 1 <= n <= SAMPLE_MAX_VOCAB:
        _fail(f"logits must be 1..65535 rows of 1..{SAMPLE_MAX_VOCAB} tokens")
    if (el != 1 and n > 1) or (b > 1 and stride < n):
        _fail("logits must have contiguous rows that do not overlap")
    if u is None or next_token is None:
        _fail("u and next_token are needed")
    _call("chr_nf4_sample_commit_batch", device, logits.data_ptr(), max(stride, n), n, b,
          _vector(u, b, device, _F32, "u"), _vector(temperature, b, device, _F32, "temperature"),
          _vector(top_k, b, device, _I32, "top_k"), _vector(top_p, b, device, _F32, "top_p"),
          _vector(min_p, b, device, _F32, "min_p"), _vector(prob, b, device, _F32, "prob"),
          _vector(next_token, b, device, _I64, "next_token"), _vector(token, b, device, _I64, "token"),
          _vector(position, b, device, _I64, "position"), _vector(finished, b, device, _U8, "finished"), int(eos))
