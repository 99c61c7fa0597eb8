"""Greedy generation for many sequences at once over the paged KV cache (uwc_b200.paged).

`PagedBatch` serves a DetQwen3's weights to sequences of different lengths that come and go: prompts are
prefilled together in chunks, a decode step is one captured CUDA graph for whatever the slots hold then,
drafted tokens are verified several at a time, and long sequences may keep a sliding window with sinks.
The reference decodes one batch of equal lengths (runtime/detrt/qwen3.py:315-329); DetQwen3.generate_greedy
is that, bit for bit. Here the linears, norms, SwiGLU and the greedy head are the same kernels, while the
keys and values are held 8-bit a page and attention is computed in floating point: repeatable, but not
detrt's bits.

A layer:
  det_rmsnorm + quant_act                        detgpu.rmsnorm_quant
  q | k | v linear, bf16 rows                    ops.gemm_epi
  head norms, rotation, keys and values to pages paged.append
  attention over the pages                       paged.attention
  o linear + residual                            ops.quant_rows_had, detgpu.linear_resid
  MLP + residual                                 detgpu.mlp_residual
"""
from __future__ import annotations

import torch

from . import detgpu, ops, paged
from ._lib import UWCError


class PagePool:
    """Which sequence holds which pages: a free list and the slots' rows of page ids (-1: none)."""

    def __init__(self, pages: int, slots: int, width: int, page_size: int):
        self.page_size, self.width = page_size, width
        self.free = list(range(pages - 1, -1, -1))
        self.rows: list[list[int]] = [[] for _ in range(slots)]

    def missing(self, slot: int, tokens: int) -> int:
        """Pages that `slot` lacks to hold `tokens` tokens."""
        return max(0, -(-tokens // self.page_size) - len(self.rows[slot]))

    def hold(self, slot: int, tokens: int) -> bool:
        """Gives `slot` pages for `tokens` tokens; True when it took any."""
        n = self.missing(slot, tokens)
        if len(self.rows[slot]) + n > self.width:
            raise ValueError(f"{tokens} tokens: a sequence holds at most {self.width * self.page_size}")
        if n > len(self.free):
            raise UWCError(f"{n} pages wanted, {len(self.free)} free: release a sequence first")
        for _ in range(n):
            self.rows[slot].append(self.free.pop())
        return n > 0

    def give_back(self, slot: int) -> None:
        self.free.extend(reversed(self.rows[slot]))
        self.rows[slot] = []

    def table(self) -> torch.Tensor:
        """(slots, width) int32, -1 past a sequence's pages."""
        return torch.tensor([r + [-1] * (self.width - len(r)) for r in self.rows], dtype=torch.int32)


class PagedBatch:
    """`slots` sequences of up to max_len tokens on one DetQwen3's weights. pages: pages of a layer's pool (by
    default enough for every slot at max_len). window / sinks: as in paged.attention (DetQwen3 takes no checkpoint
    trained with a window below max_pos, so that a window here approximates a model of full attention; its hidden
    pages stay held). graph: a step is replayed as one CUDA graph. The caller serializes its calls, as for DecodeGraph."""

    def __init__(self, model, slots: int, max_len: int, pages: int | None = None, page_size: int = 64,
                 window: int | None = None, sinks: int = 0, graph: bool = True):
        if slots < 1 or not 1 <= max_len <= model.cos.shape[0]:
            raise ValueError(f"slots {slots}, max_len {max_len}: at least one, and no more than max_pos {model.cos.shape[0]}")
        self.model, self.slots, self.max_len, self.window, self.sinks = model, slots, max_len, window, sinks
        dev = model.device
        width = -(-max_len // page_size)
        pages = slots * width if pages is None else pages
        self.caches = [paged.new_cache(pages, model.Hkv, page_size, dev) for _ in model.layers]
        self.pool = PagePool(pages, slots, width, page_size)
        self.len = [-1] * slots                       # cached tokens of a slot, -1: idle
        self._table = self.pool.table().to(dev)
        self._start = torch.full((slots,), -1, dtype=torch.int32, device=dev)
        self._cu = torch.arange(slots + 1, dtype=torch.int32, device=dev)
        self._tok = torch.zeros(slots, dtype=torch.int64, device=dev)    # a slot's newest token, not cached yet
        self._graph = None
        if graph:
            self._decode()                            # every slot idle: nothing is written
            torch.cuda.synchronize(dev)
            g = torch.cuda.CUDAGraph()
            c0 = ops.launches()
            with torch.cuda.graph(g):
                self._decode()
            self.launches_per_step = ops.launches() - c0
            ops.note_graph(-self.launches_per_step)   # captured, not launched
            self._graph = g

    # ---------------------------------------------------------------- the model
    def _rows(self, ids, table, start, cu, max_new: int, max_len: int) -> torch.Tensor:
        """The last layer's output (rows, D) of the ragged batch's new tokens, which end up in the cache."""
        m = self.model
        H, Hkv, n = m.H, m.Hkv, ids.numel()
        x = m.embed[ids]
        for L, c in zip(m.layers, self.caches):
            q1, s1 = detgpu.rmsnorm_quant(x, L["in_norm"], m.eps, L["qkv"].bs)
            qkv = ops.gemm_epi(q1, L["qkv"].Wq, ops.SEPI_BF16, x_scale=s1, w_scale=L["qkv"].sw, early_w=True)
            q, k, v = qkv.view(n, H + 2 * Hkv, paged.HD).split([H, Hkv, Hkv], 1)
            norms = dict(q_norm=L["q_norm"], k_norm=L["k_norm"], eps=m.eps) if m.qk_norm else {}
            q = paged.append(k, v, c, table, start, cu, max_new, m.cos, m.sin, q=q, **norms)
            o = paged.attention(q, c, table, start, cu, max_new, max_len, scale=m.inv_sqrt_hd, window=self.window,
                                sinks=self.sinks)
            q2, s2 = ops.quant_rows_had(o.view(n, H * paged.HD), L["o"].bs)
            r1 = detgpu.linear_resid(L["o"], q2, s2, x)
            x = detgpu.mlp_residual(L["gu"], L["down"], L["post_norm"], r1, m.eps)
        return x

    def _greedy(self, x: torch.Tensor) -> torch.Tensor:
        return self.model.next_tokens(detgpu.rmsnorm(x, self.model.norm, self.model.eps))

    def _decode(self) -> None:
        """One token a slot, everything read from and left in device memory."""
        x = self._rows(self._tok, self._table, self._start, self._cu, 1, self.max_len)
        self._tok.copy_(self._greedy(x))
        self._start.add_((self._start >= 0).int())

    def _ragged(self, slots: list[int], ids: list[list[int]], at: list[int]) -> torch.Tensor:
        """_rows of ids[i] at positions at[i] and on of slots[i]."""
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.model.device)
        cu = [0]
        for t in ids:
            cu.append(cu[-1] + len(t))
        flat = torch.tensor([t for row in ids for t in row], dtype=torch.int64, device=self.model.device)
        return self._rows(flat, self._table[slots], i32(at), i32(cu), max(map(len, ids)),
                          max(a + len(t) for a, t in zip(at, ids)))

    def _check_tokens(self, rows) -> None:
        """The embedding is read on the device, where a token id past its end would fault."""
        vocab = self.model.embed.shape[0]
        for r in rows:
            if len(r) and not (0 <= min(r) and max(r) < vocab):
                raise ValueError(f"token ids {min(r)} .. {max(r)}: the model has 0 .. {vocab - 1}")

    def _hold(self, slots: list[int], tokens: list[int]) -> None:
        if sum(self.pool.missing(s, t) for s, t in zip(slots, tokens)) > len(self.pool.free):
            raise UWCError(f"not enough pages: {len(self.pool.free)} free; release a sequence first")
        if any([self.pool.hold(s, t) for s, t in zip(slots, tokens)]):
            self._table.copy_(self.pool.table())

    # ---------------------------------------------------------------- sequences
    def active(self) -> list[int]:
        return [s for s, n in enumerate(self.len) if n >= 0]

    @torch.no_grad()
    def admit(self, prompts: list[list[int]], reserve: int = 0, chunk: int = 2048) -> dict[int, int]:
        """Prefills the prompts into idle slots, `chunk` tokens of each at a time, and returns each slot's first
        greedy token. reserve: tokens to come for which pages are taken now (later ones are taken as needed)."""
        idle = [s for s, n in enumerate(self.len) if n < 0][:len(prompts)]
        if len(idle) < len(prompts):
            raise UWCError(f"{len(prompts)} prompts, {len(idle)} idle slots")
        if any(not 0 < len(p) or len(p) + reserve > self.max_len for p in prompts):
            raise ValueError(f"a prompt is empty or, with {reserve} tokens to come, longer than {self.max_len}")
        if chunk < 1 or reserve < 0:
            raise ValueError(f"chunk {chunk}, reserve {reserve}")
        self._check_tokens(prompts)
        if not prompts:
            return {}
        self._hold(idle, [len(p) + reserve for p in prompts])
        try:
            last = [None] * len(prompts)
            for c0 in range(0, max(map(len, prompts)), chunk):
                part = [i for i, p in enumerate(prompts) if len(p) > c0]
                x = self._ragged([idle[i] for i in part], [prompts[i][c0:c0 + chunk] for i in part], [c0] * len(part))
                end = 0
                for i in part:
                    end += len(prompts[i][c0:c0 + chunk])
                    last[i] = x[end - 1]
            tok = self._greedy(torch.stack(last))
        except BaseException:
            for s in idle:
                self.pool.give_back(s)
            self._table.copy_(self.pool.table())
            raise
        where = torch.tensor(idle, device=self.model.device)
        self._tok[where] = tok
        self._start[where] = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device=self.model.device)
        for s, p in zip(idle, prompts):
            self.len[s] = len(p)
        return dict(zip(idle, tok.tolist()))

    @torch.no_grad()
    def step(self) -> dict[int, int]:
        """The next greedy token of every active slot; refused while one of them holds max_len tokens."""
        act = self.active()
        if not act:
            return {}
        if max(self.len) >= self.max_len:
            raise ValueError(f"slot {self.len.index(max(self.len))} holds max_len {self.max_len} tokens")
        self._hold(act, [self.len[s] + 1 for s in act])
        if self._graph is None:
            self._decode()
        else:
            self._graph.replay()
            ops.note_graph(self.launches_per_step)
        for s in act:
            self.len[s] += 1
        tok = self._tok.tolist()
        return {s: tok[s] for s in act}

    @torch.no_grad()
    def verify(self, drafts: dict[int, list[int]]) -> dict[int, list[int]]:
        """One step for the slots of `drafts`, with tokens guessed to follow each one's newest: the greedy tokens
        that the model itself puts there, up to and with the first that differs from the guess. The cache keeps
        what was confirmed; a rejected token's place is written again by the next call (its page's scale stays as it
        grew, if it did)."""
        if not drafts:
            return {}
        slots = sorted(drafts)
        if any(not (0 <= s < self.slots and self.len[s] >= 0) for s in slots):
            raise ValueError(f"slots {slots}: not all active")
        if any(self.len[s] + 1 + len(drafts[s]) > self.max_len for s in slots):
            raise ValueError(f"a slot's drafts end past max_len {self.max_len}")
        self._check_tokens(drafts.values())
        self._hold(slots, [self.len[s] + 1 + len(drafts[s]) for s in slots])
        newest = self._tok.tolist()
        ids = [[newest[s]] + list(drafts[s]) for s in slots]
        said = self._greedy(self._ragged(slots, ids, [self.len[s] for s in slots])).tolist()
        out, r0 = {}, 0
        for s, row in zip(slots, ids):
            mine = said[r0:r0 + len(row)]
            r0 += len(row)
            n = 1
            while n < len(row) and mine[n - 1] == row[n]:
                n += 1
            out[s] = mine[:n]
            self.len[s] += n
        where = torch.tensor(slots, device=self.model.device)
        self._tok[where] = torch.tensor([out[s][-1] for s in slots], device=self.model.device)
        self._start[where] = torch.tensor([self.len[s] for s in slots], dtype=torch.int32, device=self.model.device)
        return out

    def read(self, slot: int, layer: int, first: int = 0, n: int | None = None, dtype=torch.bfloat16):
        """The layer's cached keys and values of n tokens of a slot from `first` on: two (n, Hkv, 128) tensors."""
        n = self.len[slot] - first if n is None else n
        if first < 0 or n < 0 or first + n > self.len[slot]:
            raise ValueError(f"tokens {first} .. {first + n - 1} of slot {slot}, which holds {self.len[slot]}")
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=self.model.device)
        return paged.gather(self.caches[layer], self._table[slot:slot + 1], i32([first]), i32([0, n]), n, n, dtype)

    def release(self, slot: int) -> None:
        """Ends a sequence: its slot and pages are free."""
        if self.len[slot] < 0:
            raise ValueError(f"slot {slot} is idle")
        self.pool.give_back(slot)
        self.len[slot] = -1
        self._start[slot] = -1
        self._table.copy_(self.pool.table())

    def generate(self, prompts: list[list[int]], n_new: int) -> list[list[int]]:
        """n_new greedy tokens after each prompt, from a batch whose slots are all idle: sequences enter as slots
        and pages come free. Prompts that cannot be served are refused before any is."""
        if self.active():
            raise UWCError("generate wants every slot idle")
        if n_new < 1:
            return [[] for _ in prompts]
        more = n_new - 1                              # the last token is answered, not cached
        need = [-(-(len(p) + more) // self.pool.page_size) for p in prompts]
        for i, p in enumerate(prompts):
            if len(p) == 0 or len(p) + more > self.max_len:
                raise ValueError(f"prompt {i} is empty or, with {more} tokens to cache, longer than {self.max_len}")
            if need[i] > len(self.pool.free):
                raise UWCError(f"prompt {i} needs {need[i]} pages, of {len(self.pool.free)}")
        self._check_tokens(prompts)
        out: list[list[int]] = [[] for _ in prompts]
        waiting, owner = list(range(len(prompts))), {}
        try:
            while waiting or owner:
                room, enter = len(self.pool.free), []
                while waiting and len(enter) < self.len.count(-1) and need[waiting[0]] <= room:
                    room -= need[waiting[0]]
                    enter.append(waiting.pop(0))
                got = self.admit([prompts[i] for i in enter], reserve=more)
                owner.update(zip(got, enter))
                if not got:
                    got = self.step()
                for s, t in got.items():
                    out[owner[s]].append(t)
                for s in [s for s, i in owner.items() if len(out[i]) == n_new]:
                    self.release(s)
                    del owner[s]
        finally:                                      # a call that failed leaves no slot occupied
            for s in self.active():
                self.release(s)
        return out
