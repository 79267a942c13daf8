"""The serving operators measured: rows appended to a paged KV cache with rotary positions, attention of
ragged rows (single tokens, drafted trees, prompt chunks) over that cache, and the sampled pick.

``run`` with ``own`` false computes them from elementary torch operations in 32 bits (64 for the
sampler's sums); with ``own`` true it calls ``gpu.nf4``. Head layouts are those of the framework's
decoder configurations.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

#: (n_q, n_kv, head_dim) of the framework's decoder configurations
HEADS = {"3b": (16, 2, 128), "14b": (40, 8, 128), "20b": (48, 8, 128), "medium": (8, 2, 64)}


def listed():
    return [
        # one new token of one sequence on the smallest served configuration: pure latency
        dict(name="append_token", op="append", heads="3b", batch=1, rows=1, kv_lo=1500, kv_hi=1500, page=16,
             style="half", rot=128, table="bf16", ragged=False, pad=0),
        # a decode step of 64 sequences, FP32 tables of a long-context scaling
        dict(name="append_decode_64", op="append", heads="14b", batch=64, rows=1, kv_lo=40, kv_hi=2000, page=64,
             style="half", rot=128, table="fp32", ragged=False, pad=0),
        # prompt chunks of several requests in one call; interleaved pairs on part of the head, padded tail
        dict(name="append_prompts", op="append", heads="20b", batch=7, rows=1999, kv_lo=2000, kv_hi=4000, page=32,
             style="interleaved", rot=64, table="fp32", ragged=True, pad=13),
        # one token of one sequence, the decode step's smallest attention
        dict(name="attn_token", op="attn", heads="14b", batch=1, rows=1, kv_lo=1792, kv_hi=1792, page=64,
             tree=False, ragged=False, pad=0),
        # 64 sequences of different lengths decoded together
        dict(name="attn_decode_64", op="attn", heads="14b", batch=64, rows=1, kv_lo=150, kv_hi=3500, page=16,
             tree=False, ragged=False, pad=0),
        # few sequences with very long contexts and only two kv heads
        dict(name="attn_long", op="attn", heads="3b", batch=3, rows=1, kv_lo=90001, kv_hi=131071, page=128,
             tree=False, ragged=False, pad=0),
        # small drafted trees, odd lengths
        dict(name="attn_tree_small", op="attn", heads="20b", batch=5, rows=5, kv_lo=333, kv_hi=1777, page=32,
             tree=True, ragged=True, pad=3),
        # drafted trees of 32 tokens for 16 sequences
        dict(name="attn_tree_32", op="attn", heads="14b", batch=16, rows=32, kv_lo=2100, kv_hi=6000, page=64,
             tree=True, ragged=False, pad=0),
        # prompt chunks over a cached prefix: the compute-bound end
        dict(name="attn_prompts", op="attn", heads="14b", batch=3, rows=2047, kv_lo=2100, kv_hi=4096, page=64,
             tree=False, ragged=False, pad=0),
        # one sequence's draw from the full vocabulary
        dict(name="sample_one", op="sample", batch=1, vocab=151936, masked=False, wide=False),
        # 64 sequences with their own settings, no top-k on most: the whole tail counts
        dict(name="sample_64", op="sample", batch=64, vocab=152064, masked=False, wide=True),
        # a grammar leaves a few tokens of a smaller vocabulary; odd vocabulary, rows not aligned
        dict(name="sample_masked", op="sample", batch=9, vocab=92543, masked=True, wide=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "sample"])
    if op == "sample":
        return dict(op=op, batch=_log(rng, 1, 64), vocab=_log(rng, 500, 152064), masked=rng.random() < 0.3,
                    wide=rng.random() < 0.5)
    heads = rng.choice(sorted(HEADS))
    n_q, n_kv, hd = HEADS[heads]
    page = rng.choice([16, 32, 64, 128])
    batch = _log(rng, 1, 64)
    if op == "append":
        rows = _log(rng, 1, 8192 // batch)
        kv = rows + _log(rng, 1, 2000)
        return dict(op=op, heads=heads, batch=batch, rows=rows, kv_lo=rows + (kv - rows) // 2, kv_hi=kv, page=page,
                    style=rng.choice(["half", "interleaved"]), rot=rng.choice([hd, hd, hd // 2, hd // 4]),
                    table=rng.choice(["bf16", "fp32"]), ragged=rng.random() < 0.5, pad=rng.choice([0, 0, 1, 17]))
    tree = rng.random() < 0.5
    # at most about the cache rows of the 64-sequence case and the scores of the prompt case
    rows = 1 if rng.random() < 0.35 else _log(rng, 2, 80 if tree else 2047)
    kv = _log(rng, 64, min(131071, 64 * 1800 * 8 // (batch * n_kv)))
    rows = max(1, min(rows, kv, int(3 * 2047 * 40 * 3000 / (batch * n_q * kv))))
    return dict(op=op, heads=heads, batch=batch, rows=rows, kv_lo=max(rows, kv // rng.choice([1, 2, 10])), kv_hi=kv,
                page=page, tree=tree, ragged=rng.random() < 0.5, pad=rng.choice([0, 0, 2, 31]))


# --------------------------------------------------------------------------- inputs


def _lengths(case):
    """Rows and cache rows of each sequence, spread over the case's ranges (the same for every seed)."""
    b = np.arange(case["batch"])
    f, g = (b * 0.6180339887 + 0.35) % 1.0, (b * 0.7548776662 + 0.8) % 1.0
    rows = np.full(case["batch"], case["rows"])
    if case["ragged"]:
        rows = 1 + np.floor(g * (case["rows"] - 1) + 0.5).astype(np.int64)
    kv = np.floor(case["kv_lo"] + f * (case["kv_hi"] - case["kv_lo"])).astype(np.int64)
    kv[0] = case["kv_hi"]
    return rows.astype(np.int64), np.maximum(kv, rows)


def _cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _pages(case, kv, rs, gen):
    """Pools and a table whose pages lie in no order; one page belongs to nobody."""
    _, n_kv, hd = HEADS[case["heads"]]
    per = -(-kv // case["page"])
    n_pages = int(per.sum()) + 1
    order = rs.permutation(n_pages - 1).astype(np.int32)
    table = np.zeros((len(kv), int(per.max())), np.int32)
    at = 0
    for i, p in enumerate(per):
        table[i, :p] = order[at:at + p]
        at += int(p)
    shape = (n_pages, case["page"], n_kv, hd)
    k = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    v = torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)
    return k, v, _cuda(table)


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 32))
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": dict(case)}
    if case["op"] == "sample":
        b, n = case["batch"], case["vocab"]
        # a flat body, a few dozen likely tokens with exponential gaps, bf16 as the lm_head leaves them
        x = torch.randn((b, n), generator=gen, device="cuda") * 2.0
        likely = torch.randint(0, n, (b, 48), generator=gen, device="cuda")
        gaps = torch.empty((b, 48), device="cuda").exponential_(1.0, generator=gen)
        x.scatter_reduce_(1, likely, 6.0 + 4.0 * gaps, "amax")  # the same whatever repeats among `likely`
        if case["masked"]:
            x.masked_fill_(torch.rand((b, n), generator=gen, device="cuda") > 50.0 / n, -math.inf)
            x[:, n // 2] = 1.0
        s["logits"] = x.to(torch.bfloat16)
        s["u"] = torch.rand(b, generator=gen, device="cuda")
        pick = lambda v: rs.choice(np.array(v), b)  # noqa: E731
        s["temperature"] = _cuda(pick([0.6, 0.8, 1.0, 1.2, 0.0] if b > 4 else [0.7, 1.0]).astype(np.float32))
        s["top_k"] = _cuda(pick([0, 0, 0, 2000] if case["wide"] else [1, 20, 50, 400, 0]).astype(np.int32))
        s["top_p"] = _cuda(pick([1.0, 0.9, 0.95, 0.99]).astype(np.float32))
        s["min_p"] = _cuda(pick([0.0, 0.0, 0.0, 0.02]).astype(np.float32))
        s["next"] = torch.zeros(b, dtype=torch.int64, device="cuda")
        s["prob"] = torch.zeros(b, dtype=torch.float32, device="cuda")
        return s
    n_q, n_kv, hd = HEADS[case["heads"]]
    rows, kv = _lengths(case)
    t = int(rows.sum()) + case["pad"]
    s["k_pages"], s["v_pages"], s["page_table"] = _pages(case, kv, rs, gen)
    seq = np.full(t, -1, np.int32)
    slot = np.zeros(t, np.int64)
    at = 0
    for i, (r, l) in enumerate(zip(rows, kv)):
        seq[at:at + r] = i
        slot[at:at + r] = np.arange(l - r, l)
        at += int(r)
    if case["op"] == "append":
        # the stacked q/k/v product, whose row views the append takes
        y = torch.randn((t, (n_q + 2 * n_kv) * hd), generator=gen, device="cuda", dtype=torch.bfloat16)
        s["q"], s["k"], s["v"] = y[:, :n_q * hd], y[:, n_q * hd:(n_q + n_kv) * hd], y[:, (n_q + n_kv) * hd:]
        s["seq"], s["slot"] = _cuda(seq), _cuda(slot)
        ang = np.outer(np.arange(case["kv_hi"] + 1), 1e6 ** (-np.arange(0, case["rot"], 2) / case["rot"]))
        if case["table"] == "fp32":
            ang = ang / 4.0
        s["cos"], s["sin"] = _cuda(np.cos(ang).astype(np.float32)), _cuda(np.sin(ang).astype(np.float32))
        if case["table"] == "bf16":
            s["cos"], s["sin"] = s["cos"].bfloat16(), s["sin"].bfloat16()
        s["q_out"] = torch.zeros((t, n_q, hd), dtype=torch.bfloat16, device="cuda")
        return s
    s["q"] = 1.5 * torch.randn((t, n_q, hd), generator=gen, device="cuda", dtype=torch.bfloat16)
    s["kv_len"] = _cuda(kv.astype(np.int32))
    s["q_start"] = _cuda(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32))
    s["scale"] = hd ** -0.5
    s["tree"] = None
    if case["tree"]:
        words = -(-case["rows"] // 64)
        bits = np.zeros((t, words), np.uint64)
        at = 0
        for r in rows:  # a random tree: each draft hangs on an earlier one
            for i in range(int(r)):
                if i:
                    bits[at + i] = bits[at + rs.randint(max(0, i - 6), i)]
                bits[at + i, i // 64] |= np.uint64(1) << np.uint64(i % 64)
            at += int(r)
        s["tree"] = _cuda(bits.view(np.int64))
    s["out"] = torch.zeros((t, n_q * hd), dtype=torch.bfloat16, device="cuda")
    return s


# --------------------------------------------------------------------------- the operators


def _nf4():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "deep-fold_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import gpu.nf4

    return gpu.nf4


_OPS = None


def run(s):
    global _OPS
    op = s["case"]["op"]
    if own:
        if _OPS is None:
            _OPS = _nf4()
        if op == "append":
            q = _OPS.nf4_rope_kv_paged(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["page_table"], s["cos"],
                                       s["sin"], s["slot"], seq=s["seq"], interleaved=s["case"]["style"] == "interleaved",
                                       q_out=s["q_out"])
            return {"q": q, "k": s["k_pages"], "v": s["v_pages"]}
        if op == "attn":
            return _OPS.nf4_attn_paged(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["kv_len"], s["scale"],
                                       q_start=s["q_start"], tree=s["tree"], out=s["out"])
        _OPS.nf4_sample_commit_batch(s["logits"], s["u"], s["next"], temperature=s["temperature"], top_k=s["top_k"],
                                     top_p=s["top_p"], min_p=s["min_p"], prob=s["prob"])
        return {"token": s["next"], "prob": s["prob"]}
    if op == "append":
        return _append_plain(s)
    return _attn_plain(s) if op == "attn" else _sample_plain(s)


def _rotate(x, c, sn, rot, interleaved):
    """x [t, heads, hd] float32, c / sn [t, 1, rot/2]."""
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * c - b * sn, b * c + a * sn), dim=-1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat((a * c - b * sn, b * c + a * sn), dim=-1)
    return torch.cat((y, x[..., rot:]), dim=-1)


def _append_plain(s):
    n_pages, page, n_kv, hd = s["k_pages"].shape
    t, rot = s["q"].shape[0], 2 * s["cos"].shape[1]
    inter = s["case"]["style"] == "interleaved"
    live = s["seq"] >= 0
    row = s["page_table"][s["seq"].clamp(min=0).long(), s["slot"] // page].long() * page + s["slot"] % page
    row = torch.where(live, row, n_pages * page - 1)  # a skipped row puts back what the page of nobody holds
    c, sn = s["cos"][s["slot"]].float()[:, None], s["sin"][s["slot"]].float()[:, None]
    k = _rotate(s["k"].reshape(t, n_kv, hd).float(), c, sn, rot, inter).to(torch.bfloat16)
    kp, vp = s["k_pages"].view(-1, n_kv, hd), s["v_pages"].view(-1, n_kv, hd)
    keep = live[:, None, None]
    kp[row] = torch.where(keep, k, kp[row])
    vp[row] = torch.where(keep, s["v"].reshape(t, n_kv, hd), vp[row])
    q = _rotate(s["q"].reshape(t, -1, hd).float(), c, sn, rot, inter).to(torch.bfloat16)
    s["q_out"].copy_(torch.where(keep, q, s["q_out"]))
    return {"q": s["q_out"], "k": s["k_pages"], "v": s["v_pages"]}


def _attn_plain(s):
    n_pages, page, n_kv, hd = s["k_pages"].shape
    t, n_q = s["q"].shape[:2]
    case, dev = s["case"], s["q"].device
    b, n, longest = case["batch"], case["rows"], case["kv_hi"]
    rep = n_q // n_kv
    used = s["page_table"][:, :-(-longest // page)].long()
    k = s["k_pages"][used].view(b, -1, n_kv, hd).float()
    v = s["v_pages"][used].view(b, -1, n_kv, hd).float()
    l = k.shape[1]
    start, count = s["q_start"][:-1].long(), s["q_start"].diff().long()
    i = torch.arange(n, device=dev)
    at = (start[:, None] + i).clamp(max=t - 1)                                    # [b, n]
    q = s["q"][at].float().view(b, n, n_kv, rep, hd).permute(0, 2, 1, 3, 4).reshape(b, n_kv, n * rep, hd)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)) * s["scale"]                       # [b, n_kv, n*rep, l]
    length = s["kv_len"].long()
    j = torch.arange(l, device=dev) - (length - count)[:, None]                   # [b, l]: draft number of a cache row
    if s["tree"] is None:
        seen = j[:, None, :] <= i[None, :, None]
    else:
        words = s["tree"].shape[1]
        jj = j.clamp(0, 64 * words - 1)[:, None, :].expand(b, n, l)
        seen = ((torch.gather(s["tree"][at], 2, jj >> 6) >> (jj & 63)) & 1).bool() & (j < 64 * words)[:, None, :]
        seen = seen | (j < 0)[:, None, :]
    seen = (seen & (torch.arange(l, device=dev) < length[:, None])[:, None, :])   # [b, n, l]
    x = x.view(b, n_kv, n, rep, l).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(x.sub_(m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(b, n_kv, n * rep, l), v.permute(0, 2, 1, 3)).view(b, n_kv, n, rep, hd)
    o = (o / torch.where(total > 0, total, 1.0)).permute(0, 2, 1, 3, 4).reshape(b, n, n_q * hd).to(torch.bfloat16)
    row = torch.arange(t, device=dev)
    owner = torch.searchsorted(s["q_start"][1:].long(), row, right=True)
    live = owner < b
    owner = owner.clamp(max=b - 1)
    s["out"].copy_(torch.where(live[:, None], o[owner, (row - start[owner]).clamp(0, n - 1)], s["out"]))
    return s["out"]


def _sample_plain(s):
    x = s["logits"].double()
    b, n = x.shape
    greedy = (s["temperature"] <= 0)[:, None]
    temp = torch.where(greedy, 1.0, s["temperature"][:, None].double())
    x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / temp)
    j = torch.arange(n, device=x.device)
    n_k = torch.where(s["top_k"] > 0, s["top_k"], n).clamp(max=n)[:, None]
    w = torch.where(j < n_k, w, 0.0)
    cum = torch.cumsum(w, 1)
    before = cum - w
    before[:, 1:] = cum[:, :-1]
    keep = (before < s["top_p"][:, None].double() * cum[:, -1:]) | (s["top_p"][:, None] >= 1)
    keep = (keep & (w >= s["min_p"][:, None].double()) & (j < n_k)) | (j == 0)
    keep = keep & (~greedy | (j == 0))
    last = keep.sum(1, keepdim=True) - 1
    total = cum.gather(1, last)
    r = s["u"][:, None].double() * total
    at = torch.minimum((cum <= r).sum(1, keepdim=True), last)
    s["next"].copy_(order.gather(1, at)[:, 0])
    s["prob"].copy_((w.gather(1, at) / total)[:, 0])
    return {"token": s["next"], "prob": s["prob"]}


# --------------------------------------------------------------------------- what cannot be avoided


def work(case):
    if case["op"] == "sample":
        n = case["batch"] * case["vocab"]
        return {"bytes": 2 * n + 32 * case["batch"], "flops": n}
    n_q, n_kv, hd = HEADS[case["heads"]]
    rows, kv = _lengths(case)
    t = int(rows.sum())
    if case["op"] == "append":
        one = (n_q + 2 * n_kv) * hd * 2
        return {"bytes": t * (2 * one + case["rot"] * (4 if case["table"] == "fp32" else 2) + 16),
                "flops": 3 * t * (n_q + n_kv) * case["rot"]}
    prefix = (kv - rows) * rows
    inside = rows * (rows + 1) // 2 if not case["tree"] else rows * np.minimum(rows, 6)
    return {"bytes": int(kv.sum()) * n_kv * hd * 4 + 2 * t * n_q * hd * 2 + t * 8 * (-(-case["rows"] // 64)) * case["tree"],
            "flops": 4 * n_q * hd * int((prefix + inside).sum())}


# --------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return {"token": None, "prob": _sample_exact(s)}
    n_q, n_kv, hd = HEADS[case["heads"]]
    rows, kv = _lengths(case)
    page, table = case["page"], s["page_table"].cpu().numpy()
    starts = np.concatenate([[0], np.cumsum(rows)])
    if case["op"] == "append":
        half = case["rot"] // 2
        first = [2 * i if case["style"] == "interleaved" else i for i in range(half)]
        second = [2 * i + 1 if case["style"] == "interleaved" else i + half for i in range(half)]
        turned = {}
        cos, sin = s["cos"].double()[s["slot"]], s["sin"].double()[s["slot"]]
        for name, heads in (("q", n_q), ("k", n_kv)):
            z = s[name].double().reshape(-1, heads, hd).clone()
            unit = torch.complex(cos, sin)[:, None, :]
            w = torch.complex(z[..., first].contiguous(), z[..., second].contiguous()) * unit
            z[..., first], z[..., second] = w.real, w.imag
            turned[name] = z
        turned["v"] = s["v"].double().reshape(-1, n_kv, hd)
        k, v = s["k_pages"].double(), s["v_pages"].double()
        for i in range(case["batch"]):
            lo, r = int(starts[i]), int(rows[i])
            slots = np.arange(kv[i] - r, kv[i])
            pg, off = _cuda(table[i, slots // page].astype(np.int64)), _cuda(slots % page)
            k[pg, off], v[pg, off] = turned["k"][lo:lo + r], turned["v"][lo:lo + r]
        turned["q"][int(starts[-1]):] = 0
        return {"q": turned["q"], "k": k, "v": v}
    out = torch.zeros((s["q"].shape[0], n_q, hd), dtype=torch.float64, device="cuda")
    for i in range(case["batch"]):
        lo, r, l = int(starts[i]), int(rows[i]), int(kv[i])
        pg = _cuda(table[i, :-(-l // page)].astype(np.int64))
        k = s["k_pages"][pg].reshape(-1, n_kv, hd)[:l].double()
        v = s["v_pages"][pg].reshape(-1, n_kv, hd)[:l].double()
        hide = torch.zeros((r, l), dtype=torch.bool, device="cuda")
        if s["tree"] is None:
            hide[:, l - r:] = torch.ones((r, r), dtype=torch.bool, device="cuda").triu(1)
        else:
            bits = s["tree"][lo:lo + r].cpu().numpy().view(np.uint8)
            hide[:, l - r:] = _cuda(np.unpackbits(bits, axis=1, bitorder="little")[:, :r] == 0)
        for h in range(n_q):
            x = (s["q"][lo:lo + r, h].double() @ k[:, h // (n_q // n_kv)].T) * s["scale"]
            out[lo:lo + r, h] = torch.softmax(x.masked_fill(hide, -math.inf), 1) @ v[:, h // (n_q // n_kv)]
    return out.flatten(1)


def _sample_exact(s):
    """The probability of the drawn token, one row at a time on the host."""
    got = []
    for i, x in enumerate(s["logits"].double().cpu().numpy()):
        temp, k, p, least, u = (float(s[n][i]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        x = np.sort(x[np.isfinite(x)])[::-1]
        if temp <= 0:
            got.append(1.0)
            continue
        w = np.exp((x - x[0]) / temp)[: int(k) if k > 0 else None]
        kept = w
        if p < 1:
            kept = w[: 1 + int(np.searchsorted(np.cumsum(w), p * math.fsum(w), side="left"))]
        kept = kept[kept >= least] if least <= 1 else kept[:1]
        at = int(np.searchsorted(np.cumsum(kept), u * math.fsum(kept), side="right"))
        got.append(kept[min(at, len(kept) - 1)] / math.fsum(kept))
    return torch.tensor(got, dtype=torch.float64)
