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
