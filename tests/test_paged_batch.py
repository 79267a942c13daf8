"""The paged serving path: page bookkeeping, tree masks and scaled rotary tables (CPU), and the
operators together in a decoder over a paged cache (GPU)."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from gpu.decodev2 import MEDIUM_LLAMA, TINY_INTERNLM, PagedKV, Sampling, rope_tables_scaled, tree_depths, tree_masks


def test_pages_are_handed_out_taken_back_and_never_shared():
    kv = PagedKV(MEDIUM_LLAMA, 3, 7, page=16, max_seq=64, device="cpu")
    kv.reserve(0, 17)
    kv.reserve(1, 16)
    kv.reserve(2, 33)
    held = sum(kv.owned, [])
    assert len(held) == len(set(held)) == 6 and kv.free_pages == 1
    for b in range(3):
        n = len(kv.owned[b])
        assert kv.table[b, :n].tolist() == kv.owned[b] and (kv.table[b, n:] == -1).all()
    kv.reserve(0, 5)                                     # nothing to do
    with pytest.raises(RuntimeError, match="out of cache pages"):
        kv.reserve(1, 48)
    assert kv.free_pages == 1 and len(kv.owned[1]) == 1  # a refused call takes nothing
    kv.release(2, 17)
    assert len(kv.owned[2]) == 2 and kv.free_pages == 2 and kv.table[2, 2:].tolist() == [-1, -1]
    kv.reserve(1, 48)
    kv.release(1)
    assert kv.owned[1] == [] and kv.free_pages == 3
    with pytest.raises(ValueError, match="max_seq"):
        kv.reserve(0, 65)
    for bad in (dict(page=8), dict(page=24), dict(page=0)):
        with pytest.raises(ValueError):
            PagedKV(MEDIUM_LLAMA, 1, 4, max_seq=64, device="cpu", **bad)


def test_tree_masks_hold_ancestors_and_self():
    trees = [[-1, 0, 0, 1, -1], [], [-1] + list(range(70))]
    m = tree_masks(trees)
    assert tuple(m.shape) == (5 + 71, 2)
    seen = [[j for j in range(128) if (int(w[j // 64]) >> (j % 64)) & 1] for w in m]
    assert seen[:5] == [[0], [0, 1], [0, 2], [0, 1, 3], [4]]
    assert seen[5:] == [list(range(i + 1)) for i in range(71)]
    assert tree_depths(trees[0]) == [0, 1, 1, 2, 0]
    for bad in ([0], [-1, 1], [-2], [-1, 5]):
        with pytest.raises(ValueError):
            tree_masks([bad])


@pytest.mark.parametrize("scaling", ["none", "linear", "ntk", "yarn"])
def test_scaled_tables_follow_their_formulas(scaling):
    n, rot, theta, f, orig = 5000, 64, 1e4, 4.0, 1024
    cos, sin = rope_tables_scaled(n, rot, theta, scaling=scaling, factor=f, original=orig, device="cpu")
    assert cos.dtype is torch.float32 and tuple(cos.shape) == (n, rot // 2)
    for i in (0, 1, 7, 15, 20, 31):
        inv, gain = theta ** (-2 * i / rot), 1.0
        if scaling == "linear":
            inv /= f
        elif scaling == "ntk":
            inv = (theta * f ** (rot / (rot - 2))) ** (-2 * i / rot)
        elif scaling == "yarn":
            keep = min(max((orig * inv / (2 * math.pi) - 1) / 31, 0), 1)
            inv, gain = inv * keep + inv / f * (1 - keep), 1 + 0.1 * math.log(f)
        for p in (0, 1, 333, 4999):
            # rounded to float32 once; the angle's own binary64 error is below 1e-11
            assert abs(float(cos[p, i]) - gain * math.cos(p * inv)) <= 2.0**-24 * gain + 1e-10
            assert abs(float(sin[p, i]) - gain * math.sin(p * inv)) <= 2.0**-24 * gain + 1e-10
    for bad in (dict(scaling="other"), dict(scaling="yarn"), dict(factor=0.5)):
        with pytest.raises(ValueError):
            rope_tables_scaled(8, 64, 1e4, device="cpu", **bad)
    with pytest.raises(ValueError):
        rope_tables_scaled(8, 3, 1e4, device="cpu")


def test_sampling_settings_broadcast():
    s = Sampling.of(3, "cpu", temperature=0.5, top_k=[1, 2, 3])
    assert s.temperature.tolist() == [0.5] * 3 and s.top_k.tolist() == [1, 2, 3] and s.top_p is None
    assert s.top_k.dtype is torch.int32
    with pytest.raises(ValueError):
        Sampling.of(3, "cpu", top_p=[0.1, 0.2])


# --------------------------------------------------------------------------- together, on the GPU
def _weights(spec, seed=0):
    from gpu.decodev2 import DeviceWeights, build

    return DeviceWeights.from_synth(build(spec, seed), "cuda", torch.bfloat16)


def _close(got, want):
    """The same decoder through other kernels: the executor's tolerance for logits, 5 % of the largest."""
    return float((got.float() - want.float()).abs().max()) <= 0.05 * float(want.float().abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [MEDIUM_LLAMA, TINY_INTERNLM])
def test_paged_prompts_and_steps_agree_with_the_dense_cache(spec):
    from gpu.decodev2 import DecodeState, PagedBatch, consume_prompt, teacher_force_token

    weights = _weights(spec)
    prompts = [[1, 3, 5, 7, 2, 4, 6], [2], [9, 8, 7, 6]]
    batch = PagedBatch(weights, 3, 8, page=16, max_seq=16)
    got = [batch.append([p[:3] for p in prompts], last_only=True)]           # two ragged chunks
    got.append(batch.append([p[3:] for p in prompts], last_only=True))       # sequence 1 has no rows here
    want = []
    dense = [DecodeState.allocate(spec, weights.embed) for _ in prompts]
    for st, p in zip(dense, prompts):
        consume_prompt(st, weights, p)
        want.append(st.arena.logits[0].clone())
    assert _close(got[1][0], want[0]) and _close(got[0][1], want[1]) and _close(got[1][1], want[2])
    assert batch.lens == [7, 1, 4]
    for t in (5, 6, 7):
        batch.token.fill_(t)
        batch.step()
        for b, st in enumerate(dense):
            teacher_force_token(st, weights, t)
    again = batch.append([[3], [3], [3]])
    for b, st in enumerate(dense):
        teacher_force_token(st, weights, 3)
        assert _close(again[b], st.arena.logits[0])


@pytest.mark.gpu
def test_drafted_trees_give_each_path_its_own_logits_and_accept_keeps_one():
    from gpu.decodev2 import PagedBatch

    weights = _weights(MEDIUM_LLAMA)
    prompts = [[1, 3, 5, 7], [9, 8]]
    drafts, trees = [[4, 5, 6, 7, 8], [3, 2, 1]], [[-1, 0, 0, 1, 2], [-1, 0, 0]]
    batch = PagedBatch(weights, 2, 8, page=16, max_seq=32)
    batch.append(prompts)
    logits = batch.append(drafts, trees=trees)
    assert batch.lens == [4, 2]
    row = 0
    for b in range(2):
        for i in range(len(drafts[b])):
            path, j = [], i
            while j >= 0:
                path.insert(0, drafts[b][j])
                j = trees[b][j]
            one = PagedBatch(weights, 1, 4, page=16, max_seq=32)
            want = one.append([prompts[b] + path])[-1]
            assert _close(logits[row], want), (b, i)
            row += 1
    # keep 4 -> 6 -> 8 and 3 -> 1, then go on: as if only those had been appended
    batch.accept(0, [0, 2, 4], 5)
    batch.accept(1, [0, 2], 3)
    assert batch.lens == [7, 4]
    got = batch.append([[11], [12]])
    for b, seq in enumerate(([1, 3, 5, 7, 4, 6, 8, 11], [9, 8, 3, 1, 12])):
        one = PagedBatch(weights, 1, 4, page=16, max_seq=32)
        assert _close(got[b], one.append([seq])[-1])
    with pytest.raises(ValueError):
        batch.accept(0, [2, 1], 3)


@pytest.mark.gpu
def test_generation_greedy_and_sampled():
    from gpu.decodev2 import PagedBatch
    from gpu.decodev2.batch import BatchLoop

    weights = _weights(MEDIUM_LLAMA)
    prompts = [[1, 3, 5, 7], [4, 5, 6], [9, 8, 7, 6, 5, 4]]
    u = torch.rand((8, 3), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    batch = PagedBatch(weights, 3, 12, page=16, max_seq=32)
    greedy = batch.generate(prompts, 8, chunk=4)
    cold = Sampling.of(3, temperature=0.0)
    assert batch.generate(prompts, 8, chunk=4, sampling=cold, u=u) == greedy
    warm = Sampling.of(3, temperature=[1.0, 2.0, 0.7], top_k=[0, 5, 40], top_p=0.95, min_p=0.01)
    first = batch.generate(prompts, 8, chunk=4, sampling=warm, u=u)
    assert batch.generate(prompts, 8, chunk=4, sampling=warm, u=u) == first  # the draws are given
    assert first != greedy and all(0 <= t < MEDIUM_LLAMA.vocab for s in first for t in s)
    # over the dense cache: temperature 0 is its greedy stream, and the draws are its logits' own
    loop = BatchLoop(weights, 3)
    assert loop.generate(prompts, 8, sampling=cold, u=u) == loop.generate(prompts, 8)
    streams = loop.generate(prompts, 8, sampling=warm, u=u)
    assert loop.generate(prompts, 8, sampling=warm, u=u) == streams
    with pytest.raises(ValueError, match="sampling needs u"):
        loop.generate(prompts, 8, sampling=warm)
    assert np.shape(streams) == (3, 8)


@pytest.mark.gpu
def test_the_step_of_a_paged_batch_captured():
    """Append, attention and draw of one layer in one graph: a replay follows the registers."""
    import paged_ref as ref
    from gpu.nf4 import nf4_attn_paged, nf4_rope_kv_paged, nf4_sample_commit_batch

    gen = torch.Generator(device="cuda").manual_seed(3)
    lens = [33, 100]
    kp, vp, table = ref.make_cache(2, [128, 128], 16, 2, 64, gen)
    y = torch.randn((2, 12 * 64), generator=gen, device="cuda").to(torch.bfloat16)
    q, k, v = y.split([8 * 64, 2 * 64, 2 * 64], dim=1)
    cos, sin = rope_tables_scaled(256, 64, 1e4, device="cuda")
    slot = torch.tensor(lens, device="cuda")
    kv_len, u = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.rand(2, device="cuda")
    out, nxt = torch.zeros((2, 512), dtype=torch.bfloat16, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")

    def body():
        kv_len.copy_(slot)
        kv_len.add_(1)
        r = nf4_rope_kv_paged(q, k, v, kp, vp, table, cos, sin, slot)
        nf4_attn_paged(r, kp, vp, table, kv_len, 0.125, out=out)
        nf4_sample_commit_batch(out, u, nxt, position=slot)

    body()
    slot.copy_(torch.tensor(lens))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    slot.copy_(torch.tensor(lens))
    seen = []
    for _ in range(3):
        y.copy_(torch.randn(y.shape, generator=gen, device="cuda"))
        u.copy_(torch.rand(2, generator=gen, device="cuda"))
        graph.replay()
        seen.append((out.clone(), nxt.clone(), y.clone(), u.clone()))
    assert slot.tolist() == [n + 3 for n in lens]
    # the same steps one by one
    slot.copy_(torch.tensor(lens))
    for want_out, want_next, rows, un in seen:
        y.copy_(rows)
        u.copy_(un)
        body()
        assert torch.equal(out, want_out) and torch.equal(nxt, want_next)
