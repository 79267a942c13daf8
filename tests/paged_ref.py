"""64-bit restatements of the paged-cache ops and the sampled pick, used by their tests."""

from __future__ import annotations

import math

import numpy as np
import torch


def make_cache(batch, lens, page, n_kv, hd, gen, device="cuda", spare=2, poison=True, strided=False):
    """Pools whose pages lie in shuffled order; rows no sequence owns hold NaN."""
    rs = np.random.RandomState(batch * 1000 + page)
    per = [max(1, -(-int(n) // page)) for n in lens]
    n_pages = sum(per) + spare
    order = rs.permutation(n_pages)
    table = np.full((batch, max(per) + 1), n_pages + 7, np.int32)  # unused entries: no page
    at = 0
    for b, p in enumerate(per):
        table[b, :p] = order[at:at + p]
        at += p
    shape = (n_pages, page, n_kv, hd)
    if strided:  # both pools in one tensor, page by page
        both = torch.full((n_pages, 2, page, n_kv, hd), math.nan, dtype=torch.bfloat16, device=device)
        k, v = both[:, 0], both[:, 1]
    else:
        k = torch.full(shape, math.nan, dtype=torch.bfloat16, device=device)
        v = torch.full(shape, math.nan, dtype=torch.bfloat16, device=device)
    for b in range(batch):
        for a in range(0, int(lens[b]), page):
            m = min(page, int(lens[b]) - a)
            pg = int(table[b, a // page])
            k[pg, :m] = torch.randn((m, n_kv, hd), generator=gen, device=device).to(torch.bfloat16)
            v[pg, :m] = torch.randn((m, n_kv, hd), generator=gen, device=device).to(torch.bfloat16)
    if not poison:
        k.nan_to_num_(0.0)
        v.nan_to_num_(0.0)
    return k, v, torch.from_numpy(table).to(device)


def rows_of(pool, table, b, length):
    page = pool.shape[1]
    return torch.stack([pool[int(table[b, a // page]), a % page] for a in range(length)]) if length else \
        torch.zeros((0,) + tuple(pool.shape[2:]), device=pool.device)


def attention(q, k_pages, v_pages, table, kv_len, q_start, scale, tree=None):
    """(out, A): the result and sum_t p_t |v_t| of every element, both float64 [T, n_q, hd]."""
    t, n_q, hd = q.shape
    n_kv = k_pages.shape[2]
    out = torch.zeros((t, n_q, hd), dtype=torch.float64)
    mag = torch.zeros_like(out)
    tab = table.cpu().numpy()
    kp, vp, qd = k_pages.double().cpu(), v_pages.double().cpu(), q.double().cpu()
    for b in range(len(kv_len)):
        r0, r1, n = q_start[b], q_start[b + 1], int(kv_len[b])
        if r1 == r0 or n == 0:
            continue
        page = kp.shape[1]
        owned = [a for a in range(n) if 0 <= tab[b, a // page] < kp.shape[0]]
        k = torch.stack([kp[tab[b, a // page], a % page] for a in owned])
        v = torch.stack([vp[tab[b, a // page], a % page] for a in owned])
        base = n - (r1 - r0)
        for i in range(r1 - r0):
            if tree is None:
                see = [x for x, a in enumerate(owned) if a - base <= i]
            else:
                words = [int(w) & (2**64 - 1) for w in tree[r0 + i].tolist()]
                bit = lambda d: d // 64 < len(words) and (words[d // 64] >> (d % 64)) & 1  # noqa: E731
                see = [x for x, a in enumerate(owned) if a < base or bit(a - base)]
            if not see:
                continue
            kk, vv = k[see], v[see]
            for h in range(n_q):
                g = h // (n_q // n_kv)
                p = torch.softmax((kk[:, g] @ qd[r0 + i, h]) * scale, 0)
                out[r0 + i, h] = p @ vv[:, g]
                mag[r0 + i, h] = p @ vv[:, g].abs()
    return out, mag


def attention_tolerance(out, mag):
    """Half a bf16 step (2^-8) on each probability - at most 2^-8 sum p|v| together - and on the
    result; the scores' and sums' float32 errors (128 products of size about 1, exp2 and the
    running sum: below 2^-11 of sum p|v|) and the second-order term ride on the first."""
    return 2.0**-8 * (1.13 * mag + 1.01 * out.abs()) + 1e-30


def rotate(x, cos, sin, interleaved):
    """(y, |a c| + |b s|) in float64 for x [T, heads, hd], cos / sin [T, rot/2]."""
    x, c, s = x.double(), cos.double()[:, None], sin.double()[:, None]
    rot = 2 * cos.shape[1]
    first = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    second = first + 1 if interleaved else first + rot // 2
    y, mag = x.clone(), torch.zeros_like(x)
    a, b = x[..., first.to(x.device)], x[..., second.to(x.device)]
    y[..., first.to(x.device)], y[..., second.to(x.device)] = a * c - b * s, b * c + a * s
    mag[..., first.to(x.device)] = (a * c).abs() + (b * s).abs()
    mag[..., second.to(x.device)] = (b * c).abs() + (a * s).abs()
    return y, mag


def rotate_tolerance(y, mag):
    """One rounding to bf16 (2^-8 of the value) after two products and a sum in float32."""
    return 2.0**-8 * y.abs() * 1.01 + 3 * 2.0**-24 * mag


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, prob) of one row of float64 logits, from the definition."""
    x = np.asarray(logits, dtype=np.float64)
    if np.isnan(x).any():
        return int(np.flatnonzero(np.isnan(x))[0]), 1.0
    if not temperature > 0 or not np.isfinite(x.max()):
        return int(np.argmax(x)), 1.0
    order = np.lexsort((np.arange(len(x)), -x))
    w = np.exp((x[order] - x.max()) / float(np.float32(temperature)))
    n = len(x) if top_k <= 0 else min(top_k, len(x))
    cum = np.cumsum(w[:n])
    keep = n
    if top_p < 1:
        before = np.concatenate([[0.0], cum[:-1]])
        keep = int((before < float(np.float32(top_p)) * cum[-1]).sum())
    if min_p > 0:
        keep = min(keep, int((w[:n] >= float(np.float32(min_p))).sum()))
    keep = max(keep, 1)
    u = min(max(float(np.float32(u)), 0.0), 1 - 2.0**-24) if u == u else 0.0
    at = min(int((cum[:keep] <= u * cum[keep - 1]).sum()), keep - 1)
    return int(order[at]), float(w[at] / cum[keep - 1])
