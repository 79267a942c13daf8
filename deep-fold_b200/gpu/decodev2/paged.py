"""Sequences over one paged KV cache: prompts, decode steps, drafted trees.

Not in the reference, whose executor reserves ``max_seq`` cache rows for its one sequence
(gpu/decodev2/kv.py:14-120). ``PagedKV`` holds the pools of all layers and hands out pages;
``PagedBatch`` runs the decoder for any rows of any of its sequences in one pass - the last
token of every sequence, a prompt chunk, or a tree of drafted tokens to be checked - on
``nf4_rope_kv_paged`` and ``nf4_attn_paged``, and picks greedily or with ``Sampling``. The
linears are those of ``batch.py``. Single GPU.
"""

from __future__ import annotations

from collections.abc import Sequence

import torch

from gpu.nf4 import (nf4_attn_paged, nf4_attn_paged_status, nf4_pick_commit_batch, nf4_rms_rows, nf4_rope_kv_paged,
                     nf4_sample_commit_batch, nf4_silu_mul)

from .batch import Sampling, _linear
from .embed import gather_embed
from .linear import DeviceWeights
from .rope import rope_tables_scaled

__all__ = ["PagedBatch", "PagedKV", "tree_depths", "tree_masks"]


def tree_depths(parents: Sequence[int]) -> list[int]:
    """Depth of every draft of a tree; ``parents[i]`` is an earlier draft, or -1 for a root."""
    depth: list[int] = []
    for i, p in enumerate(parents):
        if not -1 <= p < i:
            raise ValueError(f"draft {i} hangs on {p}, which is not an earlier draft or -1")
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def tree_masks(trees: Sequence[Sequence[int]], device=None) -> torch.Tensor:
    """The masks ``nf4_attn_paged`` takes for one tree per sequence: int64 ``[drafts, words]``,
    a draft seeing its ancestors and itself."""
    words = max(1, max((len(t) + 63) // 64 for t in trees))
    out = torch.zeros((sum(len(t) for t in trees), words), dtype=torch.int64)
    at = 0
    for parents in trees:
        tree_depths(parents)
        for i, p in enumerate(parents):
            if p >= 0:
                out[at + i] = out[at + p]
            bit = 1 << (i % 64)
            out[at + i, i // 64] |= bit - (1 << 64) if bit >> 63 else bit
        at += len(parents)
    return out.to(device) if device is not None else out


class PagedKV:
    """Pools ``[layers, n_pages, page, n_kv, head_dim]`` and the page table of ``batch`` sequences
    of at most ``max_seq`` rows. Pages are handed out and taken back on the host."""

    def __init__(self, spec, batch: int, n_pages: int, *, page: int = 64, max_seq: int | None = None, device="cuda",
                 dtype: torch.dtype = torch.bfloat16) -> None:
        if batch < 1 or n_pages < 1:
            raise ValueError("a paged cache needs sequences and pages")
        if page < 16 or page & (page - 1):
            raise ValueError(f"page must be a power of two of at least 16, got {page}")
        self.page, self.max_seq = int(page), int(max_seq or spec.max_seq)
        shape = (spec.n_layers, int(n_pages), self.page, spec.n_kv, spec.head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.owned: list[list[int]] = [[] for _ in range(batch)]
        self._free = list(range(int(n_pages) - 1, -1, -1))
        self.table = torch.full((batch, -(-self.max_seq // self.page)), -1, dtype=torch.int32, device=device)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def reserve(self, seq: int, rows: int) -> None:
        """Sees to it that sequence ``seq`` has pages for ``rows`` cache rows."""
        self.reserve_all({seq: rows})

    def reserve_all(self, rows: dict[int, int]) -> None:
        """``reserve`` for several sequences (rows by sequence): all of them, or none if it raises."""
        more = {}
        for seq, n in rows.items():
            if n > self.max_seq:
                raise ValueError(f"{n} rows exceed max_seq={self.max_seq}")
            have, need = len(self.owned[seq]), -(-n // self.page)
            if need > have:
                more[seq] = have, need
        lack = sum(need - have for have, need in more.values())
        if lack > len(self._free):
            raise RuntimeError(f"out of cache pages: sequences {list(more)} need {lack}, {len(self._free)} are free")
        for seq, (have, need) in more.items():
            own = self.owned[seq]
            own.extend(self._free.pop() for _ in range(need - have))
            self.table[seq, have:need] = torch.tensor(own[have:need], dtype=torch.int32)

    def release(self, seq: int, rows: int = 0) -> None:
        """Takes back the pages of ``seq`` beyond those that ``rows`` cache rows need."""
        own, keep = self.owned[seq], -(-rows // self.page)
        if keep < len(own):
            self._free.extend(reversed(own[keep:]))
            del own[keep:]
            self.table[seq, keep:] = -1


class PagedBatch:
    """``batch`` sequences over one paged cache. ``rope`` are keyword arguments of
    ``rope_tables_scaled`` (scaling for contexts longer than the weights were trained on).

    ``append``, ``step`` and ``pick`` leave their results on the device; ``check``, which ``generate``
    calls, tells whether the attention that made them ran to its end.

    Rotated queries and probabilities are bf16 here, where the dense cache's decode keeps two bf16 terms of
    each: logits differ by roundings, and tokens can where two are that close."""

    def __init__(self, weights: DeviceWeights, batch: int, n_pages: int, *, page: int = 64, max_seq: int | None = None,
                 rope: dict | None = None) -> None:
        spec = weights.spec
        if spec.tp != 1:
            raise RuntimeError("the paged cache is single-GPU")
        self.weights, self.spec, self.batch = weights, spec, int(batch)
        dev = weights.lm_head.packed.device
        self.device = dev
        self.kv = PagedKV(spec, batch, n_pages, page=page, max_seq=max_seq, device=dev)
        self.cos, self.sin = rope_tables_scaled(self.kv.max_seq, spec.head_dim, spec.rope_theta, device=dev, **(rope or {}))
        #: cache rows of every sequence, and the token each one goes on with (not in the cache yet)
        self.lens = [0] * self.batch
        self._open: list[list[int]] = [[] for _ in range(self.batch)]  # parents of the drafts behind ``lens``
        self.token = torch.zeros(self.batch, dtype=torch.int64, device=dev)
        self.prob = torch.ones(self.batch, dtype=torch.float32, device=dev)
        self._scratch = torch.zeros((self.batch, 16), dtype=torch.uint8, device=dev)

    # ------------------------------------------------------------------ the decoder
    def _forward(self, tokens: torch.Tensor, slot: torch.Tensor, kv_len: torch.Tensor, *, seq=None, position=None,
                 q_start=None, tree=None, rows: torch.Tensor | None = None) -> torch.Tensor:
        """Logits ``[rows, vocab]`` of the given rows (default: all) of a pass over ``tokens [T]``."""
        w, spec, kv = self.weights, self.spec, self.kv
        t, hd = int(tokens.numel()), spec.head_dim
        x = gather_embed(w.embed, tokens, dtype=torch.bfloat16)
        for li, layer in enumerate(w.layers):
            h = nf4_rms_rows(x, layer.norm1, spec.rms_eps)
            if layer.wqkv is None and layer.qkv_rows is not None:
                q, k, v = _linear(layer.qkv_rows, h).split([layer.q.M, layer.k.M, layer.v.M], dim=1)
            elif layer.wqkv is None:
                q, k, v = _linear(layer.q, h), _linear(layer.k, h), _linear(layer.v, h)
            else:
                y = _linear(layer.wqkv, h).view(t, spec.n_kv, spec.n_rep + 2, hd)
                q = y[:, :, : spec.n_rep].reshape(t, spec.n_q, hd)
                k, v = y[:, :, -2].contiguous(), y[:, :, -1].contiguous()
            q = nf4_rope_kv_paged(q, k, v, kv.k[li], kv.v[li], kv.table, self.cos, self.sin, slot, seq=seq,
                                  position=position)
            attn = nf4_attn_paged(q, kv.k[li], kv.v[li], kv.table, kv_len, spec.attn_scale, q_start=q_start, tree=tree)
            x = _linear(layer.o, attn, add=x)
            h = nf4_rms_rows(x, layer.norm2, spec.rms_eps)
            gu = (_linear(layer.gate_up, h) if layer.gate_up is not None
                  else torch.cat([_linear(layer.gate, h), _linear(layer.up, h)], dim=1))
            x = _linear(layer.down, nf4_silu_mul(gu, spec.intermediate), add=x)
        if rows is not None:
            x = x.index_select(0, rows)
        return _linear(w.lm_head, nf4_rms_rows(x, w.final_norm, spec.rms_eps))

    def _i64(self, v) -> torch.Tensor:
        return torch.tensor(v, dtype=torch.int64, device=self.device)

    def _i32(self, v) -> torch.Tensor:
        return torch.tensor(v, dtype=torch.int32, device=self.device)

    def append(self, rows: Sequence[Sequence[int]], *, trees: Sequence[Sequence[int]] | None = None,
               last_only: bool = False) -> torch.Tensor:
        """One pass over new rows of every sequence (none for some): prompt chunks, or with ``trees``
        (a parent list per sequence) drafted tokens. Their keys and values go to the cache rows
        behind ``lens``, which it leaves alone for drafts and advances otherwise. Returns the
        logits of all rows, in order, or of each sequence's last row (``last_only``). A call that
        raises has taken no pages."""
        if len(rows) != self.batch or not any(len(r) for r in rows):
            raise ValueError(f"need rows for {self.batch} sequences")
        if trees is not None and [len(t) for t in trees] != [len(r) for r in rows]:
            raise ValueError("a tree has one parent per draft")
        if any(len(r) and not 0 <= min(r) <= max(r) < self.spec.vocab for r in rows):
            raise ValueError(f"a token outside 0..{self.spec.vocab - 1}")
        start, seq, slot, position, kv_len = [0], [], [], [], []
        for b, r in enumerate(rows):
            n, at = len(r), self.lens[b]
            start.append(start[-1] + n)
            seq += [b] * n
            slot += range(at, at + n)
            position += range(at, at + n) if trees is None else [at + d for d in tree_depths(trees[b])]
            kv_len.append(at + n)
        self.kv.reserve_all({b: kv_len[b] for b, r in enumerate(rows) if len(r)})
        last = self._i64([e - 1 for e, r in zip(start[1:], rows) if len(r)]) if last_only else None
        logits = self._forward(self._i64([t for r in rows for t in r]), self._i64(slot), self._i32(kv_len),
                               seq=self._i32(seq), position=self._i64(position), q_start=self._i32(start),
                               tree=None if trees is None else tree_masks(trees, self.device), rows=last)
        if trees is None:
            self.lens = kv_len
        for b, r in enumerate(rows):
            if len(r):  # what was drafted there before is overwritten
                self._open[b] = [] if trees is None else list(trees[b])
        return logits

    def pick(self, logits: torch.Tensor, sampling: Sampling | None = None, u: torch.Tensor | None = None) -> torch.Tensor:
        """Every sequence's next token from ``logits [batch, vocab]`` (greedy without ``sampling``,
        else drawn with the uniform numbers ``u [batch]``), kept as ``token``."""
        if sampling is None:
            nf4_pick_commit_batch(logits, self.token, self._scratch, eos=int(self.spec.eos_id))
        else:
            nf4_sample_commit_batch(logits, u, self.token, prob=self.prob, **sampling.settings())
        return self.token

    def step(self, sampling: Sampling | None = None, u: torch.Tensor | None = None) -> torch.Tensor:
        """Feeds every sequence its ``token`` and picks the next one."""
        self.kv.reserve_all({b: n + 1 for b, n in enumerate(self.lens)})
        logits = self._forward(self.token, self._i64(self.lens), self._i32([n + 1 for n in self.lens]))
        self.lens = [n + 1 for n in self.lens]
        self._open = [[] for _ in range(self.batch)]
        return self.pick(logits, sampling, u)

    def accept(self, seq: int, path: Sequence[int], drafts: int) -> None:
        """Keeps the drafts ``path`` (indices of the sequence's ``drafts`` last appended, from a root down,
        each the child of the one before) as the sequence's next rows and drops the others."""
        at, kv, parents = self.lens[seq], self.kv, self._open[seq]
        if drafts != len(parents):
            raise ValueError(f"sequence {seq} has {len(parents)} drafts open, not {drafts}")
        up = -1
        for i in path:
            if not 0 <= i < drafts or parents[i] != up:
                raise ValueError(f"draft {i} is not {'a root' if up < 0 else f'a child of {up}'}")
            up = i
        self._open[seq] = []
        src = [at + i for i in path]
        dst = list(range(at, at + len(path)))
        if src != dst:
            where = lambda rows: (self._i64([kv.owned[seq][r // kv.page] for r in rows]),  # noqa: E731
                                  self._i64([r % kv.page for r in rows]))
            (sp, so), (dp, do) = where(src), where(dst)
            kv.k[:, dp, do] = kv.k[:, sp, so]
            kv.v[:, dp, do] = kv.v[:, sp, so]
        self.lens[seq] = at + len(path)
        kv.release(seq, self.lens[seq])

    def check(self) -> None:
        """Raises if a wait of the attention ran out since the last look: the tokens picked and the rows
        appended since are then undefined. Synchronises."""
        code = nf4_attn_paged_status(self.device)
        if code:
            raise RuntimeError(f"paged attention gave up a wait (status {code}): the results since the last check, "
                               "cache rows included, are undefined")

    def reset(self) -> None:
        for b in range(self.batch):
            self.kv.release(b)
        self.lens = [0] * self.batch
        self._open = [[] for _ in range(self.batch)]

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], n_new: int, *, sampling: Sampling | None = None,
                 u: torch.Tensor | None = None, chunk: int = 512) -> list[list[int]]:
        """``n_new`` ids per sequence (EOS ignored): the prompts in chunks, all sequences together,
        then steps. With ``sampling``, ``u [n_new, batch]`` are the uniform numbers."""
        if len(prompts) != self.batch or not all(len(p) for p in prompts):
            raise ValueError(f"need {self.batch} prompts")
        if sampling is not None and (u is None or tuple(u.shape) != (int(n_new), self.batch)):
            raise ValueError(f"sampling needs u [{int(n_new)}, {self.batch}]")
        self.reset()
        logits = torch.empty((self.batch, self.spec.vocab), dtype=torch.bfloat16, device=self.device)
        for lo in range(0, max(len(p) for p in prompts), chunk):
            rows = [list(p[lo:lo + chunk]) for p in prompts]
            got = self.append(rows, last_only=True)
            logits.index_copy_(0, self._i64([b for b, r in enumerate(rows) if r]), got)
        trace = torch.zeros((int(n_new), self.batch), dtype=torch.int64, device=self.device)
        for i in range(int(n_new)):
            ui = None if u is None else u[i]
            trace[i].copy_(self.pick(logits, sampling, ui) if i == 0 else self.step(sampling, ui))
        self.check()
        return trace.t().tolist()
