"""The sampled pick against a 64-bit restatement of its definition."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def _run(logits, u, **kw):
    from gpu.nf4 import nf4_sample_commit_batch

    b = logits.shape[0]
    nxt = torch.full((b,), -5, dtype=torch.int64, device="cuda")
    prob = torch.full((b,), -5.0, device="cuda")
    dev = {k: torch.tensor(v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda") for k, v in kw.items()}
    nf4_sample_commit_batch(logits, torch.tensor(u, dtype=torch.float32, device="cuda"), nxt, prob=prob, **dev)
    return nxt.tolist(), prob.tolist()


def _check(logits, u, **kw):
    tokens, probs = _run(logits, u, **kw)
    for i, row in enumerate(logits.double().cpu().numpy()):
        want, p = ref.sample(row, u[i], **{k: v[i] for k, v in kw.items()})
        assert tokens[i] == want, (i, tokens[i], want, {k: v[i] for k, v in kw.items()})
        assert abs(probs[i] - p) <= 2.0**-23 * p, (i, probs[i], p)  # one rounding of a 64-bit quotient


@pytest.mark.parametrize("n", [1, 2, 7, 8, 63, 1000, 4096, 4097, 32003, 92544, 151936, 300001])
def test_settings_alone_and_together(n):
    gen = torch.Generator(device="cuda").manual_seed(n)
    b = 12
    logits = (3 * torch.randn((b, n), generator=gen, device="cuda")).to(BF16)
    u = torch.rand(b, generator=gen, device="cuda").tolist()
    _check(logits, u)
    _check(logits, u, temperature=[0.3, 0.7, 1.0, 1.5, 4.0, 100.0] * 2)
    _check(logits, u, top_k=[1, 2, 3, 50, 1000, n, n + 1, 0, -1, 5, 10, 4096])
    _check(logits, u, top_p=[0.0, 1e-6, 0.1, 0.5, 0.9, 0.999, 1.0, 1.5, 0.3, 0.7, 0.99, 0.95])
    _check(logits, u, min_p=[0.0, 1e-5, 0.01, 0.1, 0.5, 0.999, 1.0, 2.0, 0.02, 0.05, 0.2, 1e-3])
    _check(logits, u, temperature=[0.8, 1.2, 0.5] * 4, top_k=[0, 40, 400, 7] * 3, top_p=[0.9, 1.0, 0.8, 0.95] * 3,
           min_p=[0.0, 0.05, 0.01] * 4)


def test_ends_of_the_unit_interval():
    gen = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn((8, 5000), generator=gen, device="cuda").to(BF16)
    u = [0.0, 1 - 2.0**-24, 1.0, 2.0, -1.0, math.nan, 0.5, 2.0**-30]
    _check(logits, u)
    _check(logits, u, top_k=[3] * 8)
    _check(logits, u, top_p=[0.4] * 8)


def test_ties_go_to_the_lowest_index():
    """Equal logits everywhere, two values only, and a tie across the top-k border."""
    b, n = 6, 70000
    flat = torch.zeros((b, n), dtype=BF16, device="cuda")
    _check(flat, [0.0, 0.25, 0.5, 0.75, 0.9999, 0.1])
    _check(flat, [0.0, 0.25, 0.5, 0.75, 0.9999, 0.1], top_k=[1, 2, 4, 8, 69999, 65536])
    _check(flat, [0.9, 0.25, 0.5, 0.75, 0.9999, 0.1], top_p=[0.5, 0.25, 0.125, 0.75, 0.5, 1.0])
    two = flat.clone()
    two[:, ::3] = 2.0
    two[:, 1::3] = -0.0
    _check(two, [0.0, 0.3, 0.6, 0.8, 0.95, 0.9999], top_k=[23334, 23335, 23336, 30000, 69999, 0])


def test_masked_rows_and_rows_that_cannot_be_drawn_from():
    """-inf everywhere, +inf, NaN: picked as the greedy pick does; -inf among finite logits has no
    weight, however large top_k is; the type's lowest value is a finite logit like any other."""
    from gpu.nf4 import nf4_pick_commit_batch

    b, n = 9, 3001
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((b, n), generator=gen, device="cuda").to(BF16)
    x[0] = -math.inf
    x[1, 2000], x[1, 2500] = math.inf, math.inf
    x[2, 77], x[2, 78] = math.nan, math.nan
    x[3] = -math.inf
    x[3, 2999] = -5.0
    x[4, 10:] = -math.inf
    x[5] = torch.finfo(BF16).min
    x[6] = torch.finfo(BF16).min
    x[6, 44] = 0.0
    x[7, :5] = torch.finfo(BF16).max
    x[8, 1], x[8, 0] = -math.nan, math.inf
    u = [0.9, 0.9, 0.5, 0.99, 0.999, 0.5, 0.999, 0.7, 0.5]
    _check(x, u)
    _check(x, u, top_k=[3, 1, 2, 100, 3000, 10, 5, 4, 0], temperature=[1.0, 2.0, 0.5, 1.0, 1.0, 3.0, 1.0, 0.1, 1.0])
    _check(x, u, temperature=[0.0, -1.0, math.nan, 1e-30, 0.0, 1e30, math.inf, 1e-38, 1.0])
    tokens, _ = _run(x, u, temperature=[0.0] * b)
    want = torch.zeros(b, dtype=torch.int64, device="cuda")
    nf4_pick_commit_batch(x, want, torch.zeros((b, 16), dtype=torch.uint8, device="cuda"))
    assert tokens == want.tolist()


def test_commit_strided_unaligned_rows_and_repeats():
    from gpu.nf4 import nf4_sample_commit_batch

    gen = torch.Generator(device="cuda").manual_seed(3)
    wide = torch.randn((33, 20011), generator=gen, device="cuda").to(BF16)
    for lo, hi in ((0, 20011), (1, 20000), (3, 9), (5, 6)):
        logits = wide[:, lo:hi]
        u = torch.rand(33, generator=gen, device="cuda").tolist()
        _check(logits, u, top_p=[0.9] * 33)
        tok, pos = torch.zeros(33, dtype=torch.int64, device="cuda"), torch.arange(33, device="cuda")
        nxt, fin = torch.zeros(33, dtype=torch.int64, device="cuda"), torch.zeros(33, dtype=torch.uint8, device="cuda")
        want, _ = _run(logits, u)
        for _ in range(2):
            nf4_sample_commit_batch(logits, torch.tensor(u, device="cuda"), nxt, token=tok, position=pos, finished=fin,
                                    eos=want[7])
        assert nxt.tolist() == want and tok.tolist() == want
        assert pos.tolist() == [i + 2 for i in range(33)]
        assert fin.tolist() == [int(t == want[7]) for t in want]


def test_draws_follow_the_distribution():
    """Uniform numbers on a grid: every token is drawn for its share of the unit interval."""
    n, b = 50, 4096
    x = torch.linspace(-2, 3, n, device="cuda").to(BF16).expand(b, n)
    tokens, _ = _run(x.contiguous(), ((np.arange(b) + 0.5) / b).tolist())
    p = torch.softmax(x[0].double().cpu(), 0).numpy()
    share = np.bincount(tokens, minlength=n) / b
    assert np.abs(share - p).max() <= 1.0 / b  # a grid of b points meets an interval b|I| +- 1 times


def test_captured_draw_follows_its_inputs():
    from gpu.nf4 import nf4_sample_commit_batch

    gen = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((3, 9000), generator=gen, device="cuda").to(BF16)
    u, nxt = torch.rand(3, generator=gen, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    nf4_sample_commit_batch(x, u, nxt)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nf4_sample_commit_batch(x, u, nxt)
    for _ in range(3):
        x.copy_(torch.randn((3, 9000), generator=gen, device="cuda"))
        u.copy_(torch.rand(3, generator=gen, device="cuda"))
        graph.replay()
        got = nxt.tolist()
        assert got == [ref.sample(r, float(v))[0] for r, v in zip(x.double().cpu().numpy(), u.cpu())]


def test_slices_longer_than_a_counter_counts():
    """So many rows that two blocks share a row of 151936 tokens: one value may then occur more often in
    a block's half than 16 bits count - all equal, a lowest-value mask, zeros of both signs, NaN."""
    n, b = 151936, 90
    gen = torch.Generator(device="cuda").manual_seed(9)
    logits = (2 * torch.randn((b, n), generator=gen, device="cuda")).to(BF16)
    low = torch.finfo(BF16).min
    for i in range(b):
        row = logits[i]
        kind = i % 9
        if kind == 0:
            row[:] = 1.5
        elif kind == 1:  # all masked but a few
            keep = row[::5000].clone()
            row[:] = low
            row[::5000] = keep
        elif kind == 2:  # masked behind some place in the row
            row[100 + 800 * i:] = low
        elif kind == 3:
            row[:] = 0.0
            row[::2] = -0.0
        elif kind == 4:
            row[:] = 0.0
            row[:33000] = -0.0
            row[40000:140000] = -0.0
            row[-5:] = 1.0
        elif kind == 5:
            row[: 70000 + i] = 3.0
        elif kind == 6:  # two values that take most of a half each
            row[:37000] = 2.0
            row[37000:76000] = 2.015625
            row[76000:] = -1.0
        elif kind == 7:
            row[7:] = -math.inf
    u = torch.rand(b, generator=gen, device="cuda").tolist()
    _check(logits, u)
    _check(logits, u, temperature=[0.7] * b, top_k=[(0, 40, 40000, 75000, 120000)[i % 5] for i in range(b)],
           top_p=[(1.0, 0.9, 0.5)[i % 3] for i in range(b)], min_p=[(0.0, 0.01)[i % 2] for i in range(b)])
    nans = logits.clone()
    nans[::2, 5:] = math.nan
    nans[1::2, 80000:] = -math.nan
    tokens, _ = _run(nans, u)
    assert tokens == [5 if i % 2 == 0 else 80000 for i in range(b)]
