"""The paged-cache ops and the decoder over them at the edges of what their contracts allow."""

from __future__ import annotations

import math

import pytest
import torch

import paged_ref as ref

BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,hd", [(8, 2, 64), (4, 2, 16), (10, 2, 128)])
@pytest.mark.parametrize("rows,kv,front,behind", [([1, 1], [40, 7], 1, 2), ([3, 0, 2], [40, 7, 2], 5, 0),
                                                  ([40, 21], [300, 30], 33, 1), ([0, 0], [3, 4], 4, 3)])
def test_rows_in_front_of_the_first_sequence(n_q, n_kv, hd, rows, kv, front, behind):
    """Padding in front (``q_start[0] > 0``) as behind: zero in a new result, left alone in a given one."""
    from gpu.nf4 import nf4_attn_paged

    gen = _gen(front + hd)
    kp, vp, table = ref.make_cache(len(kv), kv, 16, n_kv, hd, gen)
    starts = [front]
    for r in rows:
        starts.append(starts[-1] + r)
    t = starts[-1] + behind
    q = torch.randn((t, n_q, hd), generator=gen, device="cuda").to(BF16)
    torch.full((t, n_q * hd), math.nan, dtype=BF16, device="cuda")  # what the allocator hands out next
    got = nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.1, q_start=_i32(starts))
    want, mag = ref.attention(q, kp, vp, table, kv, starts, 0.1)  # zeros where no sequence owns the row
    assert not got[:front].any() and not got[starts[-1]:].any()
    err = (got.view(t, n_q, hd).double().cpu() - want).abs()
    assert (err <= ref.attention_tolerance(want, mag)).all()
    out = torch.full((t, n_q * hd), 3.0, dtype=BF16, device="cuda")
    nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.1, q_start=_i32(starts), out=out)
    assert (out[:front] == 3.0).all() and (out[starts[-1]:] == 3.0).all()
    assert torch.equal(out[front:starts[-1]], got[front:starts[-1]])


def test_overlap_of_rows_of_two_widths():
    """Against the elements themselves: never missed, and not reported where the steps are one."""
    from gpu.nf4.paged import _overlap

    flat = torch.empty(1000, dtype=BF16)

    def elements(t):
        first = (t.data_ptr() - flat.data_ptr()) // 2
        return set((first + torch.arange(t.shape[0])[:, None] * t.stride(0) + torch.arange(t.shape[1])).flatten().tolist())

    def both(a, b):
        args = [(t.data_ptr(), t.shape[0], t.stride(0)) for t in (a, b)]
        got = _overlap(*args[0], *args[1], a.shape[1], b.shape[1])
        assert got == _overlap(*args[1], *args[0], b.shape[1], a.shape[1])
        return got, bool(elements(a) & elements(b))

    y = flat[:600].view(6, 100)
    for a0, a1, b0, b1 in ((0, 60, 60, 80), (0, 60, 59, 80), (0, 60, 80, 100), (20, 30, 0, 20), (20, 30, 0, 21),
                           (99, 100, 0, 99), (0, 100, 50, 51), (40, 60, 45, 46)):
        got, shared = both(y[:, a0:a1], y[:, b0:b1])
        assert got == shared
        for a, b in ((y[:3, a0:a1], y[2:, b0:b1]), (y[:1, a0:a1], y[:, b0:b1]), (y[3:, a0:a1], y[:3, b0:b1])):
            got, shared = both(a, b)
            assert got or not shared
    assert both(y[:1, :60], y[:1, 60:80]) == both(y[5:, 30:], y[5:, :30]) == (False, False)
    assert both(flat[:240].view(4, 60), flat[240:300].view(3, 20)) == (False, False)
    assert both(flat[:240].view(4, 60), flat[200:260].view(3, 20)) == (True, True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3])
def test_append_refuses_to_write_over_its_inputs(rows):
    from gpu.nf4 import nf4_rope_kv_paged

    gen = _gen(2)
    kp, vp, table = ref.make_cache(3, [20, 20, 20], 16, 2, 64, gen, poison=False)
    y = torch.randn((rows, 12 * 64), generator=gen, device="cuda").to(BF16)
    q, k, v = y.split([8 * 64, 2 * 64, 2 * 64], dim=1)
    cos, sin = torch.ones((32, 32), device="cuda"), torch.zeros((32, 32), device="cuda")
    slot = torch.full((rows,), 19, device="cuda")

    def call(k, v, out, kp=kp, vp=vp):
        return nf4_rope_kv_paged(q, k, v, kp, vp, table, cos, sin, slot, q_out=out)

    other = torch.zeros_like(y)
    out, inside = other[:, :512], other[:, 448:576]     # `inside` begins in the rows given for q_out
    with pytest.raises(RuntimeError, match="q_out must not overlap k"):
        call(inside, v, out)
    with pytest.raises(RuntimeError, match="q_out must not overlap v"):
        call(k, inside, out)
    two = torch.zeros((kp.shape[0], 2) + tuple(kp.shape[1:]), dtype=BF16, device="cuda")
    pages = two.view((-1,) + tuple(kp.shape[1:]))
    for a, b in ((kp, kp), (two[:, 0], two[:, 0]), (pages[:6], pages[5:11])):
        with pytest.raises(RuntimeError, match="k_pages and v_pages must not overlap"):
            call(k, v, out, a, b)
    assert not two.any() and not other.any()
    assert call(k, v, q) is q                           # q, k and v side by side in one product
    call(k, v, out, two[:, 0], two[:, 1])               # the pools' pages in turn
    page = table[:rows, 1].long()
    assert torch.equal(two[page, 1, 3].flatten(1), v) and torch.equal(two[page, 0, 3].flatten(1), k)


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,hd,rows,kv", [
    (8, 1, 128, [1, 1, 1], [2000, 5, 700]), (40, 8, 128, [1] * 64, [33 * i + 1 for i in range(64)]),
    (4, 2, 64, [4, 0, 3], [900, 7, 64]), (4, 2, 16, [30, 1], [3000, 9]), (6, 1, 32, [3, 1], [40, 20000])])
def test_thin_waits_that_run_out_say_so_and_the_call_ends(n_q, n_kv, hd, rows, kv):
    """With no polls at all the first copy not there yet is given up: a status, a call that returns
    with nothing in flight, and an ordinary call behind it as right as ever."""
    from gpu.nf4 import _lib, nf4_attn_paged, nf4_attn_paged_status

    lib = _lib.load()
    gen = _gen(hd + len(rows))
    kp, vp, table = ref.make_cache(len(kv), kv, 16, n_kv, hd, gen)
    table[0, 1] = -1                                    # a block that is not copied among those that are
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    q = torch.randn((starts[-1], n_q, hd), generator=gen, device="cuda").to(BF16)
    call = lambda: nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.1, q_start=_i32(starts))  # noqa: E731
    want = call()
    assert nf4_attn_paged_status() == 0
    lib.chr_nf4_set_attn_paged_polls(0)
    try:
        for _ in range(3):
            call()
            assert nf4_attn_paged_status() == 20
            assert nf4_attn_paged_status() == 0         # read and cleared
    finally:
        lib.chr_nf4_set_attn_paged_polls(-1)
    for _ in range(3):
        assert torch.equal(call(), want)
    assert nf4_attn_paged_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,n_kv,hd,rows,kv,page,tree", [
    (10, 2, 128, [52, 51], [700, 51], 64, False), (8, 2, 64, [103, 40, 0, 77], [1031, 400, 9, 77], 32, False),
    (16, 1, 128, [300], [2300], 512, False), (40, 8, 128, [32] * 16, [2100 + 100 * i for i in range(16)], 64, True),
    (5, 1, 64, [600, 30], [9000, 400], 16, False)])
def test_wide_waits_that_run_out_say_so_and_the_call_ends(n_q, n_kv, hd, rows, kv, page, tree):
    """As for the thin form: whichever role gives up first, copies and products in flight are waited for."""
    from gpu.nf4 import _lib, nf4_attn_paged, nf4_attn_paged_status

    lib = _lib.load()
    gen = _gen(hd + len(rows))
    kp, vp, table = ref.make_cache(len(kv), kv, page, n_kv, hd, gen)
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    q = torch.randn((starts[-1], n_q, hd), generator=gen, device="cuda").to(BF16)
    mask = None
    if tree:
        mask = torch.tensor([[(2 << i) - 1] for r in rows for i in range(r)], device="cuda")
    call = lambda: nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.1, q_start=_i32(starts), tree=mask)  # noqa: E731
    want = call()
    assert nf4_attn_paged_status() == 0
    try:
        for polls in (0, 0, 1):
            lib.chr_nf4_set_attn_paged_polls(polls)
            got = call()
            status = nf4_attn_paged_status()
            assert 1 <= status <= 12 if polls == 0 else 0 <= status <= 12
            if status == 0:
                assert torch.equal(got, want)           # every wait was over in time
            assert nf4_attn_paged_status() == 0
    finally:
        lib.chr_nf4_set_attn_paged_polls(-1)
    for _ in range(3):
        assert torch.equal(call(), want)
    assert nf4_attn_paged_status() == 0


def _weights(spec, seed=0):
    from gpu.decodev2 import DeviceWeights, build

    return DeviceWeights.from_synth(build(spec, seed), "cuda", BF16)


@pytest.mark.gpu
def test_generation_raises_when_the_attention_gave_up():
    """The tokens of a run in which a wait ran out are not handed out; the next run is as ever."""
    from gpu.decodev2 import MEDIUM_LLAMA, PagedBatch
    from gpu.nf4 import _lib, nf4_attn_paged_status

    lib = _lib.load()
    batch = PagedBatch(_weights(MEDIUM_LLAMA), 2, 8, page=16, max_seq=32)
    prompts = [[1, 3, 5, 7], [9, 8]]
    want = batch.generate(prompts, 5)
    lib.chr_nf4_set_attn_paged_polls(0)
    try:
        with pytest.raises(RuntimeError, match="gave up a wait"):
            batch.generate(prompts, 5)
        batch.append([[1], [2]])
        with pytest.raises(RuntimeError, match="gave up a wait"):
            batch.check()
    finally:
        lib.chr_nf4_set_attn_paged_polls(-1)
    batch.check()                                       # said once
    assert batch.generate(prompts, 5) == want
    assert nf4_attn_paged_status() == nf4_attn_paged_status(0) == nf4_attn_paged_status(batch.device) == 0


@pytest.mark.gpu
def test_accept_takes_a_chain_of_children_only():
    """From a root down, each draft the child of the one before, of the drafts appended last."""
    from gpu.decodev2 import MEDIUM_LLAMA, PagedBatch

    batch = PagedBatch(_weights(MEDIUM_LLAMA), 2, 8, page=16, max_seq=32)
    batch.append([[1, 3, 5, 7], [9, 8]])
    tree = [[-1, 0, 0, 1, 2, -1], [-1, -1]]
    batch.append([[4, 5, 6, 7, 8, 9], [3, 2]], trees=tree)
    before = [list(batch.lens), [list(o) for o in batch.kv.owned]]
    for path in ([1], [0, 3], [0, 1, 2], [0, 1, 4], [1, 3], [0, 5], [6], [-1], [0, 0], [3, 1]):
        with pytest.raises(ValueError):
            batch.accept(0, path, 6)
    for drafts in (5, 7, 0):
        with pytest.raises(ValueError):
            batch.accept(0, [0, 1], drafts)
    assert [list(batch.lens), [list(o) for o in batch.kv.owned]] == before
    batch.accept(0, [0, 2, 4], 6)
    with pytest.raises(ValueError):          # its drafts are settled
        batch.accept(0, [0, 2, 4], 6)
    batch.accept(1, [1], 2)
    assert batch.lens == [7, 3]
    batch.append([[4], [5, 6]], trees=[[-1], [-1, 0]])
    batch.accept(1, [], 2)                   # none kept
    assert batch.lens == [7, 3]
    batch.append([[2], [2]])                 # takes the rows of sequence 0's open draft
    with pytest.raises(ValueError):
        batch.accept(0, [0], 1)
    batch.append([[4], []], trees=[[-1], []])
    batch.token.fill_(1)
    batch.step()                             # so does a step
    with pytest.raises(ValueError):
        batch.accept(0, [0], 1)


@pytest.mark.gpu
def test_a_refused_append_or_step_takes_nothing():
    from gpu.decodev2 import MEDIUM_LLAMA, PagedBatch

    batch = PagedBatch(_weights(MEDIUM_LLAMA), 2, 3, page=16, max_seq=40)
    batch.append([list(range(1, 17)), [2]])
    state = lambda: (list(batch.lens), [list(o) for o in batch.kv.owned], batch.kv.free_pages,  # noqa: E731
                     batch.kv.table.tolist())
    before = state()
    refused = [(RuntimeError, "out of cache pages", dict(rows=[[1], [1] * 16])),
               (ValueError, "max_seq", dict(rows=[[1], [1] * 40])),
               (ValueError, "draft", dict(rows=[[1], [1]], trees=[[-1], [0]])),
               (ValueError, "token", dict(rows=[[1], [MEDIUM_LLAMA.vocab]])),
               (ValueError, "token", dict(rows=[[-1], [1]])),
               (ValueError, "one parent", dict(rows=[[1], [1]], trees=[[-1]]))]
    for kind, what, kw in refused:
        with pytest.raises(kind, match=what):
            batch.append(**kw)
        assert state() == before
    batch.append([[], [3] * 15])
    before = state()
    with pytest.raises(RuntimeError, match="out of cache pages"):  # both need a page, one is left
        batch.step()
    assert state() == before


def test_pages_for_several_sequences_or_for_none():
    from gpu.decodev2 import MEDIUM_LLAMA, PagedKV

    kv = PagedKV(MEDIUM_LLAMA, 3, 5, page=16, max_seq=64, device="cpu")
    kv.reserve_all({0: 16, 2: 20})
    state = lambda: ([list(o) for o in kv.owned], kv.free_pages, kv.table.tolist())  # noqa: E731
    before = state()
    assert [len(o) for o in before[0]] == [1, 0, 2] and before[1] == 2
    for kind, what, rows in ((RuntimeError, "out of cache pages", {0: 17, 1: 1, 2: 33}),
                             (ValueError, "max_seq", {0: 17, 1: 65}), (ValueError, "max_seq", {1: 65, 0: 17})):
        with pytest.raises(kind, match=what):
            kv.reserve_all(rows)
        assert state() == before
    kv.reserve_all({0: 17, 1: 16, 2: 32})
    assert [len(o) for o in kv.owned] == [2, 1, 2] and kv.free_pages == 0
    assert sorted(sum(kv.owned, [])) == [0, 1, 2, 3, 4]
    for b in range(3):
        n = len(kv.owned[b])
        assert kv.table[b, :n].tolist() == kv.owned[b] and (kv.table[b, n:] == -1).all()


@pytest.mark.parametrize("rot,theta,factor,original", [(128, 1e6, 4.0, 32768), (64, 1e4, 8.0, 4096)])
def test_yarn_ramp_over_pairs(rot, theta, factor, original):
    """The blend of released checkpoints, its borders found by bisection over the turns of a pair."""
    from gpu.decodev2 import rope_tables_scaled

    def index_of(turns):
        lo, hi = 0.0, float(rot)
        for _ in range(200):
            mid = (lo + hi) / 2
            lo, hi = (mid, hi) if original * theta ** (-2 * mid / rot) / (2 * math.pi) > turns else (lo, mid)
        return lo

    first, last = math.floor(index_of(32)), math.ceil(index_of(1))
    if rot == 128:
        assert (first, last) == (23, 40)
    args = dict(scaling="yarn", factor=factor, original=original, device="cpu", dtype=torch.float64)
    cos, sin = rope_tables_scaled(64, rot, theta, ramp="pairs", **args)
    gain = 1 + 0.1 * math.log(factor)
    for i in range(rot // 2):
        share = min(max((i - first) / (last - first), 0.0), 1.0)     # of the divided angle
        inv = theta ** (-2 * i / rot) * (1 - share + share / factor)
        for p in (0, 1, 63):
            assert abs(float(cos[p, i]) - gain * math.cos(p * inv)) <= 1e-12
            assert abs(float(sin[p, i]) - gain * math.sin(p * inv)) <= 1e-12
    assert not torch.equal(cos, rope_tables_scaled(64, rot, theta, ramp="turns", **args)[0])
    assert torch.equal(rope_tables_scaled(64, rot, theta, **args)[0], rope_tables_scaled(64, rot, theta, ramp="turns", **args)[0])


def test_yarn_ramps_at_their_ends():
    from gpu.decodev2 import rope_tables_scaled

    args = dict(scaling="yarn", factor=4.0, device="cpu", dtype=torch.float64)
    # every pair turns often: none is slowed; every pair turns less than once: all are but the first,
    # at which both borders, drawn to the pairs there are, then lie
    for original, slowed in ((10**9, [1.0] * 8), (4, [1.0] + [4.0] * 7)):
        cos, sin = rope_tables_scaled(9, 16, 100.0, original=original, ramp="pairs", **args)
        for i in range(8):
            inv = 100.0 ** (-2 * i / 16) / slowed[i]
            assert abs(float(sin[8, i]) - (1 + 0.1 * math.log(4.0)) * math.sin(8 * inv)) <= 1e-12
    with pytest.raises(ValueError, match="ramp"):
        rope_tables_scaled(8, 64, 1e4, original=1024, ramp="other", **args)
    with pytest.raises(ValueError, match="ramp"):
        rope_tables_scaled(8, 64, 1.0, original=1024, ramp="pairs", **args)


def test_attention_refuses_caches_whose_rows_pass_32_bits():
    """The C entry's checks need no GPU: places a few tiles behind the last cache row are still counted in
    32 bits, so a table that reaches to 2^31 rows is refused."""
    import ctypes

    from gpu.nf4 import _lib

    def call(max_pages, page):
        pages = _lib.ChrNf4Pages(k=4096, v=4096, table=4096, k_page_stride=page * 128, v_page_stride=page * 128,
                                 table_stride=max_pages, n_pages=8, page=page, n_kv=2, hd=64, batch=2, max_pages=max_pages)
        args = _lib.ChrNf4AttnPaged(pages=pages, q=4096, q_stride=512, out=4096, q_start=4096, kv_len=4096, T=3, n_q=8,
                                    scale=0.1, ws=4096, ws_floats=0)
        return _lib.load().chr_nf4_attn_paged(ctypes.byref(args), None)

    assert call((1 << 27) - 1, 16) == -3 and call((1 << 15) - 1, 65536) == -7
    assert call((1 << 27) - 512, 16) == -3 and call((1 << 27) - 513, 16) == -7   # past the rows: the workspace's check
