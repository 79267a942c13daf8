"""Paged-cache append and attention against 64-bit restatements of the same formulas."""

from __future__ import annotations

import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _i64(v):
    return torch.tensor(v, dtype=torch.int64, device="cuda")


# --------------------------------------------------------------------------- append
def _tables(n, half, dtype, gen):
    ang = torch.rand((n, half), generator=gen, device="cuda", dtype=torch.float64) * 6.28
    return torch.cos(ang).to(dtype), torch.sin(ang).to(dtype)


@pytest.mark.parametrize("n_q,n_kv,hd,rot,page", [(16, 2, 128, 128, 16), (40, 8, 128, 64, 64), (4, 2, 16, 16, 16),
                                                  (8, 2, 64, 32, 32), (3, 3, 10, 6, 16), (5, 1, 24, 4, 16),
                                                  (6, 2, 128, 2, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, BF16])
def test_append_rotates_and_writes_the_rows_and_nothing_else(n_q, n_kv, hd, rot, page, interleaved, dtype):
    from gpu.nf4 import nf4_rope_kv_paged

    gen = _gen(n_q * hd + rot)
    lens = [3 * page, page + 1, 5]
    kp, vp, table = ref.make_cache(3, lens, page, n_kv, hd, gen, poison=False)
    # sequence, slot, position: a chunk across a page border, one row at a page's start, padding,
    # a slot past the table, an entry that is no page, a position past the tables
    seq = [0, 0, 0, 1, -1, 2, 3, 0, 2, 1]
    slot = [page - 1, page, page + 1, page, 0, 4, 0, 10**9, 2 * page, 3]
    pos = [7, 8, 9, 0, 3, 60, 1, 2, 3, 64]
    good = [0, 1, 2, 3, 5]
    t = len(seq)
    y = torch.randn((t, (n_q + 2 * n_kv) * hd), generator=gen, device="cuda").to(BF16)
    q, k, v = y.split([n_q * hd, n_kv * hd, n_kv * hd], dim=1)
    cos, sin = _tables(64, rot // 2, dtype, gen)
    k0, v0 = kp.clone(), vp.clone()
    out = torch.full((t, n_q, hd), 5.0, dtype=BF16, device="cuda")
    got = nf4_rope_kv_paged(q, k, v, kp, vp, table, cos, sin, _i64(slot), seq=_i32(seq), position=_i64(pos),
                            interleaved=interleaved, q_out=out)
    assert got is out
    p = torch.tensor(pos)[good]
    want_q, mag_q = ref.rotate(q.reshape(t, n_q, hd)[good].cpu(), cos.cpu()[p], sin.cpu()[p], interleaved)
    want_k, mag_k = ref.rotate(k.reshape(t, n_kv, hd)[good].cpu(), cos.cpu()[p], sin.cpu()[p], interleaved)
    assert ((out[good].double().cpu() - want_q).abs() <= ref.rotate_tolerance(want_q, mag_q)).all()
    skipped = [i for i in range(t) if i not in good]
    assert (out[skipped] == 5.0).all()
    for i, r in enumerate(good):
        pg, off = int(table[seq[r], slot[r] // page]), slot[r] % page
        assert ((kp[pg, off].double().cpu() - want_k[i]).abs() <= ref.rotate_tolerance(want_k[i], mag_k[i])).all()
        assert torch.equal(vp[pg, off], v[r].view(n_kv, hd))
        kp[pg, off], vp[pg, off] = k0[pg, off], v0[pg, off]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    # a new q: skipped rows are zero, the others the same bits; in place: the same bits
    again = nf4_rope_kv_paged(q, k, v, kp, vp, table, cos, sin, _i64(slot), seq=_i32(seq), position=_i64(pos),
                              interleaved=interleaved)
    assert torch.equal(again[good], out[good]) and not again[skipped].any()
    keep = q.clone()
    nf4_rope_kv_paged(q, k, v, kp, vp, table, cos, sin, _i64(slot), seq=_i32(seq), position=_i64(pos),
                      interleaved=interleaved, q_out=q)
    assert torch.equal(q.reshape(t, n_q, hd)[good], out[good]) and torch.equal(q[skipped], keep[skipped])


def test_append_defaults_strided_pools_and_the_dense_paths_tables():
    """One row per sequence, positions from the slots, no q, bf16 tables as column views, pools
    whose pages are interleaved in one tensor."""
    from gpu.decodev2.rope import rope_tables_torch
    from gpu.nf4 import nf4_rope_kv_paged

    gen = _gen(3)
    n_kv, hd, page = 2, 64, 16
    kp, vp, table = ref.make_cache(4, [40, 17, 1, 33], page, n_kv, hd, gen, poison=False, strided=True)
    k = torch.randn((4, n_kv, hd), generator=gen, device="cuda").to(BF16)
    v = torch.randn((4, n_kv, hd), generator=gen, device="cuda").to(BF16)
    cos, sin = rope_tables_torch(64, hd, 1e4, device="cuda", dtype=BF16)
    slot = [39, 16, 0, 20]
    assert nf4_rope_kv_paged(None, k, v, kp, vp, table, cos[:, :hd // 2], sin[:, :hd // 2], _i64(slot)) is None
    want, mag = ref.rotate(k.cpu(), cos.cpu()[slot, :hd // 2], sin.cpu()[slot, :hd // 2], False)
    for b, a in enumerate(slot):
        pg = int(table[b, a // page])
        assert ((kp[pg, a % page].double().cpu() - want[b]).abs() <= ref.rotate_tolerance(want[b], mag[b])).all()
        assert torch.equal(vp[pg, a % page], v[b])


def test_append_unaligned_rows_give_the_same_bits():
    from gpu.nf4 import nf4_rope_kv_paged

    gen = _gen(4)
    n_q, n_kv, hd = 8, 2, 64
    base = torch.randn((300, (n_q + 2 * n_kv) * hd + 3), generator=gen, device="cuda").to(BF16)
    cos, sin = _tables(512, 16, torch.float32, gen)
    slot, seq = _i64(list(range(150)) * 2), _i32([0] * 150 + [1] * 150)
    outs = []
    for y in (base[:, 1:-2], base[:, 1:-2].contiguous()):
        kp, vp, table = ref.make_cache(2, [150, 150], 32, n_kv, hd, _gen(5), poison=False)
        q, k, v = y.split([n_q * hd, n_kv * hd, n_kv * hd], dim=1)
        outs.append((nf4_rope_kv_paged(q, k, v, kp, vp, table, cos, sin, slot, seq=seq), kp, vp))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# --------------------------------------------------------------------------- attention
def _check(q, kp, vp, table, kv, starts, scale, tree=None, **kw):
    from gpu.nf4 import nf4_attn_paged

    t, n_q, hd = q.shape
    got = nf4_attn_paged(q, kp, vp, table, _i32(kv), scale, q_start=_i32(starts), tree=tree, **kw)
    want, mag = ref.attention(q, kp, vp, table, kv, starts, scale, tree)
    err = (got.view(t, n_q, hd).double().cpu() - want).abs()
    assert torch.isfinite(got).all()
    worst = (err / ref.attention_tolerance(want, mag)).max()
    assert worst <= 1.0, f"{float(worst)} of the tolerance"
    return got


def _starts(rows):
    s = [0]
    for r in rows:
        s.append(s[-1] + r)
    return s


@pytest.mark.parametrize("n_q,n_kv,hd", [(40, 8, 128), (16, 2, 128), (8, 2, 64), (4, 2, 16), (6, 3, 32), (20, 1, 128),
                                         (3, 3, 64), (33, 1, 32)])
@pytest.mark.parametrize("kv", [[1], [0, 1, 2], [127, 128, 129, 16, 15, 17], [1000], [64, 0, 700, 3]])
def test_one_token_per_sequence(n_q, n_kv, hd, kv):
    gen = _gen(sum(kv) + n_q)
    kp, vp, table = ref.make_cache(len(kv), kv, 16, n_kv, hd, gen)
    q = torch.randn((len(kv), n_q, hd), generator=gen, device="cuda").to(BF16)
    got = _check(q, kp, vp, table, kv, _starts([1] * len(kv)), hd ** -0.5)
    from gpu.nf4 import nf4_attn_paged

    assert torch.equal(got, nf4_attn_paged(q, kp, vp, table, _i32(kv), hd ** -0.5))  # q_start's default
    for b, n in enumerate(kv):
        if n == 0:
            assert not got[b].any()


@pytest.mark.parametrize("n_q,n_kv,hd", [(10, 2, 128), (8, 2, 64), (4, 2, 16), (6, 1, 32)])
@pytest.mark.parametrize("rows,kv,page", [([5], [5], 16), ([3, 0, 9, 1], [40, 7, 130, 1], 32), ([33, 64, 2], [33, 300, 2], 16),
                                          ([130], [131], 64), ([1, 40], [257, 200], 128), ([257], [520], 16)])
def test_prompt_chunks_are_causal(n_q, n_kv, hd, rows, kv, page):
    gen = _gen(sum(rows) + hd)
    kp, vp, table = ref.make_cache(len(kv), kv, page, n_kv, hd, gen)
    q = torch.randn((sum(rows), n_q, hd), generator=gen, device="cuda").to(BF16)
    _check(q, kp, vp, table, kv, _starts(rows), 0.11)


def _tree_bits(rows, words, gen, empty=()):
    """Random ancestor masks; rows in ``empty`` see no draft, not even themselves."""
    bits = []
    for r in rows:
        mine = []
        for i in range(r):
            m = 0
            if i:
                m = mine[int(torch.randint(0, i, (1,), generator=gen, device="cuda"))]
            mine.append(m | (1 << i))
        bits += [0 if (len(bits) + j) in empty else m for j, m in enumerate(mine)]
    t = torch.zeros((len(bits), words), dtype=torch.int64)
    for i, m in enumerate(bits):
        for w in range(words):
            x = (m >> (64 * w)) & (2**64 - 1)
            t[i, w] = x - 2**64 if x >= 2**63 else x
    return t.cuda()


@pytest.mark.parametrize("n_q,n_kv,hd", [(10, 2, 128), (8, 2, 64), (4, 2, 16), (16, 1, 128)])
@pytest.mark.parametrize("rows,kv,page,words", [([5], [5], 16, 1), ([4, 7, 1], [133, 64, 260], 16, 1),
                                                ([64, 3], [200, 3], 32, 1), ([70, 130], [350, 131], 64, 3),
                                                ([16, 0, 16], [500, 0, 16], 16, 1)])
def test_trees_of_drafts(n_q, n_kv, hd, rows, kv, page, words):
    gen = _gen(sum(rows) * 7 + hd)
    kp, vp, table = ref.make_cache(len(kv), kv, page, n_kv, hd, gen)
    q = torch.randn((sum(rows), n_q, hd), generator=gen, device="cuda").to(BF16)
    _check(q, kp, vp, table, kv, _starts(rows), hd ** -0.5, _tree_bits(rows, words, gen))


def test_rows_that_see_nothing_and_rows_behind_the_last_sequence():
    """Masks that leave a row empty: zeros where there is no older cache row, the older rows alone
    where there are some; bits past a short mask are clear; the padded tail stays as it was."""
    from gpu.nf4 import nf4_attn_paged

    gen = _gen(11)
    rows, kv = [6, 5], [6, 50]
    kp, vp, table = ref.make_cache(2, kv, 16, 2, 64, gen)
    t = sum(rows) + 3
    q = torch.randn((t, 8, 64), generator=gen, device="cuda").to(BF16)
    tree = torch.cat([_tree_bits(rows, 1, gen, empty={0, 3, 8}), torch.full((3, 1), -1, device="cuda")])
    out = torch.full((t, 8 * 64), 3.0, dtype=BF16, device="cuda")
    starts = _starts(rows)
    got = nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.125, q_start=_i32(starts), tree=tree, out=out)
    want, mag = ref.attention(q, kp, vp, table, kv, starts, 0.125, tree)
    err = (got[:11].view(11, 8, 64).double().cpu() - want[:11]).abs()
    assert (err <= ref.attention_tolerance(want, mag)[:11]).all()
    assert not got[0].any() and not got[3].any() and got[8].any()
    assert (got[11:] == 3.0).all()
    fresh = nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.125, q_start=_i32(starts), tree=tree)
    assert torch.equal(fresh[:11], got[:11]) and not fresh[11:].any()


def test_more_rows_than_cache_rows_and_pages_that_are_none():
    """kv_len below the row count: the first rows' own cache rows do not exist. A table entry
    outside the pool hides its rows."""
    gen = _gen(12)
    kv, rows = [3, 90], [5, 2]
    kp, vp, table = ref.make_cache(2, kv, 16, 2, 64, gen)
    q = torch.randn((7, 8, 64), generator=gen, device="cuda").to(BF16)
    got = _check(q, kp, vp, table, kv, _starts(rows), 0.125)
    assert not got[0].any() and not got[1].any() and got[2].any()
    table[1, 1], table[1, 3] = -1, kp.shape[0]
    _check(q, kp, vp, table, kv, _starts(rows), 0.125)


def test_strided_queries_and_pools():
    gen = _gen(13)
    kv, rows = [77, 140], [4, 9]
    kp, vp, table = ref.make_cache(2, kv, 16, 2, 128, gen, strided=True)
    y = torch.randn((13, 14 * 128), generator=gen, device="cuda").to(BF16)
    q = y[:, 2 * 128:12 * 128].unflatten(1, (10, 128))
    _check(q, kp, vp, table, kv, _starts(rows), 0.09)
    wide = torch.cat([table, table], dim=1)[:, :table.shape[1]]
    _check(q, kp, vp, wide, kv, _starts(rows), 0.09)


def test_large_scores_and_infinite_keys_behind_a_mask():
    gen = _gen(14)
    kv, rows = [100], [3]
    kp, vp, table = ref.make_cache(1, kv, 16, 1, 64, gen)
    q = (30 * torch.randn((3, 4, 64), generator=gen, device="cuda")).to(BF16)
    pg = int(table[0, 98 // 16])
    kp[pg, 98 % 16] = math.inf                      # draft 1 of 3, seen by nobody
    tree = torch.tensor([[1], [1], [4]], dtype=torch.int64, device="cuda")
    from gpu.nf4 import nf4_attn_paged

    got = nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.5, q_start=_i32([0, 3]), tree=tree)
    kp[pg, 98 % 16] = 0.0
    assert torch.equal(got, nf4_attn_paged(q, kp, vp, table, _i32(kv), 0.5, q_start=_i32([0, 3]), tree=tree))
    assert torch.isfinite(got).all()


def test_many_short_sequences_beside_a_long_one():
    gen = _gen(15)
    kv = [1 + (i * 7) % 40 for i in range(300)]
    kv[123] = 3000
    rows = [1] * 300
    kp, vp, table = ref.make_cache(300, kv, 16, 1, 32, gen)
    q = torch.randn((300, 2, 32), generator=gen, device="cuda").to(BF16)
    _check(q, kp, vp, table, kv, _starts(rows), 0.2)


def test_attention_captured_follows_what_the_tensors_hold():
    """A captured call replayed with other lengths, tables and queries equals an eager call."""
    from gpu.nf4 import nf4_attn_paged

    gen = _gen(16)
    kv = [130, 700]
    kp, vp, table = ref.make_cache(2, [800, 800], 32, 2, 64, gen)
    q = torch.randn((4, 8, 64), generator=gen, device="cuda").to(BF16)
    n, starts = _i32(kv), _i32([0, 1, 4])
    out = torch.zeros((4, 512), dtype=BF16, device="cuda")
    call = lambda o: nf4_attn_paged(q, kp, vp, table, n, 0.1, q_start=starts, out=o)  # noqa: E731
    call(out)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(out)
    q.copy_(q.flip(0))
    n.copy_(_i32([800, 3]))
    starts.copy_(_i32([0, 3, 4]))
    table.copy_(table.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call(None))
    assert torch.equal(out, call(None))  # and every run gives the same bits


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3])
@pytest.mark.parametrize("rows,kv", [([1, 1], [130, 40]), ([50, 33], [300, 33])])
def test_scales_of_either_sign_and_none(scale, rows, kv):
    gen = _gen(17)
    kp, vp, table = ref.make_cache(2, kv, 16, 2, 128, gen)
    q = torch.randn((sum(rows), 6, 128), generator=gen, device="cuda").to(BF16)
    _check(q, kp, vp, table, kv, _starts(rows), scale)


@pytest.mark.parametrize("n_q,n_kv,hd", [(10, 2, 128), (8, 2, 64), (16, 1, 128), (3, 3, 64)])
@pytest.mark.parametrize("rows,kv,page", [([52, 51], [700, 51], 256), ([103, 40, 0, 77], [1031, 400, 9, 77], 32),
                                          ([300], [1300], 512), ([26, 25, 27], [90, 129, 128], 16)])
@pytest.mark.parametrize("tree", [False, True])
def test_wide_items(n_q, n_kv, hd, rows, kv, page, tree):
    """Items of one and of two query tiles, pages longer and shorter than a tile, strided pools."""
    from gpu.nf4 import _lib

    gen = _gen(sum(rows) * 3 + n_q)
    kp, vp, table = ref.make_cache(len(kv), kv, page, n_kv, hd, gen, strided=True)
    q = (2 * torch.randn((sum(rows), n_q, hd), generator=gen, device="cuda")).to(BF16)
    bits = _tree_bits(rows, 5, gen, empty={1, 40}) if tree else None
    _check(q, kp, vp, table, kv, _starts(rows), hd ** -0.5, bits)
    assert _lib.load().chr_nf4_attn_paged_status() == 0


def test_wide_rows_whose_maximum_keeps_rising():
    """Scores that grow along the cache by far more than the slack of the subtracted maximum."""
    gen = _gen(18)
    kv, rows = [1500], [60]
    kp, vp, table = ref.make_cache(1, kv, 16, 2, 128, gen)
    ramp = torch.linspace(0, 6, 1500, device="cuda")
    for a in range(1500):
        kp[int(table[0, a // 16]), a % 16] = (kp[int(table[0, a // 16]), a % 16].float() * 0.2 + ramp[a]).to(BF16)
    q = torch.rand((60, 8, 128), generator=gen, device="cuda").to(BF16)
    _check(q, kp, vp, table, kv, _starts(rows), 0.3)


def test_wide_missing_pages_and_more_rows_than_cache_rows():
    gen = _gen(19)
    kv, rows = [300, 30], [40, 50]
    kp, vp, table = ref.make_cache(2, kv, 16, 2, 64, gen)
    table[0, 2], table[0, 17], table[1, 0] = -1, kp.shape[0], 1 << 30
    q = torch.randn((90, 8, 64), generator=gen, device="cuda").to(BF16)
    got = _check(q, kp, vp, table, kv, _starts(rows), 0.125)
    assert not got[40:60].any() and got[79].any()


@pytest.mark.parametrize("n_q,n_kv,hd", [(8, 1, 128), (4, 2, 64), (4, 2, 16), (6, 3, 32), (16, 1, 128), (8, 1, 64)])
@pytest.mark.parametrize("rows,kv,page", [([3, 2], [20, 90], 16), ([8, 7], [140, 7], 32), ([40, 21], [300, 30], 64),
                                          ([150, 1], [150, 9], 256)])
@pytest.mark.parametrize("tree", [False, True])
def test_what_is_not_finite_reaches_only_the_rows_that_see_it(n_q, n_kv, hd, rows, kv, page, tree):
    """Infinities and NaN in new rows: a row that does not see them keeps every bit; one that does
    has them where their element is, or everywhere if they are in the key."""
    from gpu.nf4 import nf4_attn_paged

    gen = _gen(sum(rows) + n_q)
    kp, vp, table = ref.make_cache(len(kv), kv, page, n_kv, hd, gen)
    starts = _starts(rows)
    q = torch.randn((sum(rows), n_q, hd), generator=gen, device="cuda").to(BF16)
    bits = _tree_bits(rows, 3, gen) if tree else None
    if tree:
        bits[1] = 0  # sees no draft, not even itself
    call = lambda: nf4_attn_paged(q, kp, vp, table, _i32(kv), hd ** -0.5, q_start=_i32(starts), tree=bits).view(-1, n_q, hd)
    clean = call()
    want = clean.clone()
    n_rep = n_q // n_kv
    for b, draft, pool, head, el, value in ((0, 1, vp, 0, 3, float("nan")), (0, 2, vp, n_kv - 1, hd - 1, float("inf")),
                                            (0, rows[0] // 2 + 1, vp, 0, hd // 2, -float("inf")),
                                            (1, rows[1] - 1, kp, 0, 1, float("nan")),
                                            (1, rows[1] - 1, vp, 0, 0, float("inf"))):
        if draft >= rows[b]:
            continue
        at = kv[b] - rows[b] + draft
        pool[int(table[b, at // page]), at % page, head, el] = value
        for i in range(rows[b]):
            r = starts[b] + i
            sees = draft <= i if not tree else bool((int(bits[r, draft // 64]) >> (draft % 64)) & 1)
            if sees:
                mine = want[r, head * n_rep:(head + 1) * n_rep]
                if pool is kp:
                    mine[:] = float("nan")
                else:
                    mine[:, el] += value
    got = call()
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    assert same.all(), (~same).nonzero()[:5].tolist()
    assert not torch.equal(clean, got) or tree


def test_results_that_overlap_the_queries_are_refused():
    from gpu.nf4 import nf4_attn_paged, nf4_rope_kv_paged

    gen = _gen(1)
    kp, vp, table = ref.make_cache(2, [20, 20], 16, 2, 64, gen)
    y = torch.randn((3, 8 * 64), generator=gen, device="cuda").to(BF16)
    q = y[:2]
    with pytest.raises(RuntimeError, match="overlap"):
        nf4_attn_paged(q, kp, vp, table, _i32([20, 20]), 0.1, out=y[:2])
    with pytest.raises(RuntimeError, match="overlap"):
        nf4_attn_paged(q, kp, vp, table, _i32([20, 20]), 0.1, out=y[1:])
    cos, sin = _tables(32, 32, torch.float32, gen)
    k = torch.randn((2, 2 * 64), generator=gen, device="cuda").to(BF16)
    with pytest.raises(RuntimeError, match="overlap"):
        nf4_rope_kv_paged(q, k, k, kp, vp, table, cos, sin, _i64([19, 19]), q_out=y[1:])
    assert nf4_rope_kv_paged(q, k, k, kp, vp, table, cos, sin, _i64([19, 19]), q_out=q) is q


def test_pages_shared_between_sequences():
    """Two sequences with one prefix: the same page ids in both rows of the table."""
    from gpu.nf4 import nf4_attn_paged

    gen = _gen(11)
    kp, vp, table = ref.make_cache(2, [100, 100], 16, 2, 64, gen)
    table[1, :4] = table[0, :4]
    for rows in ([1, 1], [40, 40]):
        q = torch.randn((sum(rows), 8, 64), generator=gen, device="cuda").to(BF16)
        _check(q, kp, vp, table, [100, 90], _starts(rows), 0.125)
    q[40:] = q[:40]
    table[1] = table[0]
    out = nf4_attn_paged(q, kp, vp, table, _i32([100, 100]), 0.125, q_start=_i32([0, 40, 80]))
    assert torch.equal(out[:40], out[40:])


def test_two_calls_at_once_on_two_streams():
    from gpu.nf4 import nf4_attn_paged, nf4_rope_kv_paged

    gen = _gen(12)
    jobs = []
    for rows, kv in (([1] * 6, [900, 33, 1500, 7, 64, 2000]), ([60, 3], [700, 1200])):
        kp, vp, table = ref.make_cache(len(kv), kv, 16, 2, 128, gen)
        q = torch.randn((sum(rows), 10, 128), generator=gen, device="cuda").to(BF16)
        args = (q, kp, vp, table, _i32(kv), 0.09)
        jobs.append((args, dict(q_start=_i32(_starts(rows))), nf4_attn_paged(*args, q_start=_i32(_starts(rows)))))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    outs = [[], []]
    for _ in range(10):
        for i, (args, kw, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                outs[i].append(nf4_attn_paged(*args, **kw))
    torch.cuda.synchronize()
    for i, (_, _, want) in enumerate(jobs):
        assert all(torch.equal(o, want) for o in outs[i])
    # the append, on a stream that fills its input first
    kp, vp, table = ref.make_cache(1, [64], 16, 2, 64, gen)
    cos, sin = _tables(64, 32, torch.float32, gen)
    with torch.cuda.stream(streams[0]):
        k = torch.ones((1 << 12, 1 << 12), device="cuda").matmul(torch.ones((1 << 12, 1 << 12), device="cuda"))[:1, :128].to(BF16)
        nf4_rope_kv_paged(None, k, k, kp, vp, table, cos, sin, _i64([5]))
    streams[0].synchronize()
    assert (vp[int(table[0, 0]), 5] == 4096).all()


def test_offsets_past_32_bits():
    """Pools of more than 2^31 elements: the pages used lie at their ends."""
    from gpu.nf4 import nf4_attn_paged, nf4_rope_kv_paged

    page, n_kv, hd = 64, 2, 128
    n_pages = (1 << 31) // (page * n_kv * hd) + 40
    gen = _gen(13)
    kp = torch.empty((n_pages, page, n_kv, hd), dtype=BF16, device="cuda")
    vp = torch.empty((n_pages, page, n_kv, hd), dtype=BF16, device="cuda")
    rows = [130, 70]
    table = torch.arange(n_pages - 1, n_pages - 9, -1, dtype=torch.int32, device="cuda").view(2, 4).contiguous()
    cos, sin = _tables(256, 64, torch.float32, gen)
    k, v = (torch.randn((200, n_kv * hd), generator=gen, device="cuda").to(BF16) for _ in range(2))
    seq = _i32([0] * 130 + [1] * 70)
    slot = _i64(list(range(130)) + list(range(70)))
    nf4_rope_kv_paged(None, k, v, kp, vp, table, cos, sin, slot, seq=seq)
    small_k, small_v = kp[-8:].clone(), vp[-8:].clone()
    small_table = table - (n_pages - 8)
    for new in ([1, 1], [100, 60]):
        q = torch.randn((sum(new), 8, hd), generator=gen, device="cuda").to(BF16)
        kw = dict(q_start=_i32(_starts(new)))
        got = nf4_attn_paged(q, kp, vp, table, _i32(rows), 0.09, **kw)
        assert torch.equal(got, nf4_attn_paged(q, small_k, small_v, small_table, _i32(rows), 0.09, **kw))
        want, mag = ref.attention(q, small_k, small_v, small_table, rows, _starts(new), 0.09)
        assert ((got.view_as(q).double().cpu() - want).abs() <= ref.attention_tolerance(want, mag)).all()
