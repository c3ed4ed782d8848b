"""Ring-buffer sliding-window KV cache on the GPU.

Same constructor, attributes and six methods as the reference ``KVCache``
(inference/kv_cache.py:4-68): storage ``k, v [L, B, H, W, D]``, token ``p`` of the sequence
lives in row ``p % W``, ``t`` counts committed tokens.  ``view`` / ``write`` /
``bulk_write_packed`` keep the reference's shapes and ordering; in addition ``ring(layer)``
hands the in-place ring to the decode kernel so the per-token chronological copy that
``view`` makes once the ring has wrapped is never needed on the hot path.

:class:`B200PagedKVCache` serves sequences of uneven length: one pool of pages instead of a ring per batch row.
"""
from __future__ import annotations

from typing import Iterable, List

import torch

from . import ops


def ring_segment(t: int, staged: bool, W: int):
    """Host-side index arithmetic of ``view`` (inference/kv_cache.py:27-35): returns ``(first_pos, n)``
    -- the n = min(t + staged, W) most recent tokens start at sequence position ``first_pos``."""
    m = t + (1 if staged else 0)
    n = min(m, W)
    return m - n, n


class B200KVCache:
    def __init__(self, L, B, H, W, D, device, dtype=torch.bfloat16):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("B200KVCache lives in GPU memory; daisy_b200 has no CPU path")
        self.L, self.B, self.H, self.W, self.D = L, B, H, W, D
        self.device, self.dtype = dev, dtype
        self.reset_history()

    def reset_history(self):
        shape = (self.L, self.B, self.H, self.W, self.D)
        self.k = torch.zeros(shape, device=self.device, dtype=self.dtype)
        self.v = torch.zeros(shape, device=self.device, dtype=self.dtype)
        self.t = 0
        # the same counter in device memory, for decode launches that must not depend on host values
        # (CUDA-graph replays); kept in step with `t` by stream-ordered updates, never read back
        self.t_dev = torch.zeros(1, device=self.device, dtype=torch.int64)
        self._staged = [False] * self.L

    # ------------------------------------------------------------------ reference API
    def view(self, layer):
        """Chronological ``(k, v)`` as ``[B, n, H, D]`` (inference/kv_cache.py:26-42).  A view of the
        ring when the rows are contiguous, otherwise a gathered copy."""
        first, n = ring_segment(self.t, self._staged[layer], self.W)
        if n == 0:
            return self.k[layer, :, :, :0].transpose(1, 2), self.v[layer, :, :, :0].transpose(1, 2)
        start = first % self.W
        if start + n <= self.W:
            return (self.k[layer, :, :, start:start + n].transpose(1, 2),
                    self.v[layer, :, :, start:start + n].transpose(1, 2))
        k = torch.empty(self.B, self.H, n, self.D, device=self.device, dtype=self.dtype)
        v = torch.empty_like(k)
        ops.ring_copy_rows(self.k[layer], k, first, to_ring=False)
        ops.ring_copy_rows(self.v[layer], v, first, to_ring=False)
        return k.transpose(1, 2), v.transpose(1, 2)

    def write(self, layer, k_new, v_new):
        """Stage the new token's row at slot ``t % W`` (inference/kv_cache.py:44-51); accepts
        ``[B,1,H,D]`` or ``[B,H,1,D]``."""
        if k_new.size(1) == 1:
            k_new, v_new = k_new.transpose(1, 2), v_new.transpose(1, 2)
        k_new = k_new.to(self.dtype)
        v_new = v_new.to(self.dtype)
        if k_new.stride(-1) != 1:
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
        ops.ring_copy_rows(self.k[layer], k_new, self.t, to_ring=True)
        ops.ring_copy_rows(self.v[layer], v_new, self.t, to_ring=True)
        self._staged[layer] = True

    def advance(self):
        self.t += 1
        self.t_dev += 1
        self._staged = [False] * self.L

    def bulk_write_packed(self, kv, pos):
        """Fill from prefill output ``kv [2, L, B, H, T, D]``: the last ``min(pos, W-1)`` rows go to
        slots ``p % W`` (inference/kv_cache.py:57-68)."""
        r = min(pos, max(self.W - 1, 0))
        if r > 0:
            k, v = kv[0].to(self.dtype), kv[1].to(self.dtype)
            for layer in range(self.L):
                ops.ring_copy_rows(self.k[layer], k[layer][:, :, pos - r:pos], pos - r, to_ring=True)
                ops.ring_copy_rows(self.v[layer], v[layer][:, :, pos - r:pos], pos - r, to_ring=True)
        self.t = pos
        self.t_dev.fill_(pos)
        self._staged = [False] * self.L

    def bulk_write_layer(self, layer, k, v, pos):
        """One layer of ``bulk_write_packed`` straight from that layer's prefill output ``k, v [B,H,T,D]`` (any
        strides): the runner fills the ring layer by layer and never builds the stacked ``[2,L,B,H,T,D]`` tensor
        (models/daisy/daisy_core.py:358-369).  Call :meth:`set_position` once after the last layer."""
        r = min(pos, max(self.W - 1, 0))
        if r > 0:
            ops.ring_copy_rows(self.k[layer], k.to(self.dtype)[:, :, pos - r:pos], pos - r, to_ring=True)
            ops.ring_copy_rows(self.v[layer], v.to(self.dtype)[:, :, pos - r:pos], pos - r, to_ring=True)

    def set_position(self, pos):
        self.t = pos
        self.t_dev.fill_(pos)
        self._staged = [False] * self.L

    # ------------------------------------------------------------------ in-place access for the decode kernel
    def ring(self, layer):
        """``(k_ring, v_ring)`` as ``[B, H, W, D]`` views of the storage (no copy)."""
        return self.k[layer], self.v[layer]

    def mark_written(self, layer):
        """Record that the decode kernel stored the new row of ``layer`` itself."""
        self._staged[layer] = True


class B200PagedKVCache:
    """Keys and values of up to ``max_seqs`` sequences of uneven length in one pool of pages.

    Storage ``k, v [L, pages, H, page, D]``; position ``p`` of the sequence in slot ``s`` lies in row ``p % page`` of page
    ``table[s, p // page]`` (int32, -1: none).  ``lens [max_seqs]`` (int32 on the device, mirrored in ``length``) counts the
    tokens in the cache, -1 marks a free slot.  The kernels (``ops.paged_append``, ``paged_decode_step``, ``paged_attend``) read both on
    the device; the page bookkeeping is host arithmetic, with a copy to the device only where a row of the table changes.
    Lengths only grow: a caller that may reject stored tokens (drafts) keeps lengths and table itself."""

    def __init__(self, L, pages, H, D, max_seqs, max_len, device, dtype=torch.bfloat16, page=64):
        dev = torch.device(device)
        if dev.type != "cuda":
            raise ValueError("B200PagedKVCache lives in GPU memory; daisy_b200 has no CPU path")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"pages hold bfloat16 or float16, not {dtype}")
        if page not in (16, 32, 64, 128, 256):
            raise ValueError(f"pages hold 16, 32, 64, 128 or 256 rows, got {page}")
        self.L, self.pages, self.H, self.D = L, pages, H, D
        self.max_seqs, self.max_len, self.page = max_seqs, max_len, page
        self.device, self.dtype = dev, dtype
        shape = (L, pages, H, page, D)
        self.k = torch.zeros(shape, device=dev, dtype=dtype)
        self.v = torch.zeros(shape, device=dev, dtype=dtype)
        self.table = torch.full((max_seqs, -(-max_len // page)), -1, device=dev, dtype=torch.int32)
        self.lens = torch.full((max_seqs,), -1, device=dev, dtype=torch.int32)
        self.active = torch.zeros(max_seqs, device=dev, dtype=torch.int32)
        self.book = PageBook(pages, max_seqs, max_len, page)

    @property
    def length(self) -> List[int]:
        return self.book.length

    def layer(self, layer):
        """``(k, v)`` of one layer as ``[pages, H, page, D]`` views of the storage."""
        return self.k[layer], self.v[layer]

    def claim(self) -> int:
        """A free slot for a new sequence, of length 0."""
        slot = self.book.claim()
        self.lens[slot] = 0
        self.active[slot] = 1
        return slot

    def release(self, slot: int) -> None:
        """Give a sequence's pages back and free its slot."""
        self.book.release(slot)
        self.table[slot] = -1
        self.lens[slot] = -1
        self.active[slot] = 0

    def reserve(self, slots: Iterable[int], tokens) -> None:
        """Pages for ``tokens`` (a number, or one for each slot) more tokens of every sequence; raises ``RuntimeError``, with
        nothing changed, where the pool has too few (``ValueError`` where a sequence would outgrow its row of the table)."""
        slots = list(slots)
        counts = [tokens] * len(slots) if isinstance(tokens, int) else list(tokens)
        self._store(self.book.reserve(slots, counts))

    def forget(self, slot: int, before: int) -> None:
        """Give back the pages that hold only positions below ``before`` (a window has moved past them)."""
        self._store(self.book.forget(slot, before))

    def advance(self, slots: Iterable[int], tokens) -> None:
        """Count ``tokens`` (a number, or one for each slot) stored tokens; raises ``ValueError``, with nothing changed, where a sequence
        has no pages for them."""
        slots = list(slots)
        counts = [tokens] * len(slots) if isinstance(tokens, int) else list(tokens)
        self.book.advance(slots, counts)
        self.lens.copy_(torch.tensor(self.book.length, dtype=torch.int32))

    def _store(self, rows) -> None:
        for slot in rows:
            self.table[slot].copy_(torch.tensor(self.book.table[slot], dtype=torch.int32))


class PageBook:
    """Which pages belong to which sequence: the host side of :class:`B200PagedKVCache`, no tensors."""

    def __init__(self, pages, max_seqs, max_len, page):
        self.page, self.max_len = page, max_len
        self.free = list(range(pages - 1, -1, -1))
        self.length = [-1] * max_seqs
        self.table = [[-1] * -(-max_len // page) for _ in range(max_seqs)]
        self.first = [0] * max_seqs             # entries below have been given back
        self.end = [0] * max_seqs               # entries from here on have no page yet

    def claim(self):
        if -1 not in self.length:
            raise RuntimeError("all slots of the paged cache are taken")
        slot = self.length.index(-1)
        self.length[slot] = 0
        return slot

    def _check(self, slot):
        if not 0 <= slot < len(self.length) or self.length[slot] < 0:
            raise ValueError(f"slot {slot} holds no sequence")

    def release(self, slot):
        self._check(slot)
        row = self.table[slot]
        self.free.extend(row[self.first[slot]:self.end[slot]])
        self.table[slot] = [-1] * len(row)
        self.length[slot], self.first[slot], self.end[slot] = -1, 0, 0

    def _tokens(self, slots, counts):
        """Tokens by slot (one that comes twice has both counts), each with room in the table."""
        if len(slots) != len(counts):
            raise ValueError(f"{len(counts)} counts for {len(slots)} slots")
        tokens = {}
        for slot, n in zip(slots, counts):
            self._check(slot)
            tokens[slot] = tokens.get(slot, 0) + n
            if n < 0 or self.length[slot] + tokens[slot] > self.max_len:
                raise ValueError(f"slot {slot}: {self.length[slot]} + {tokens[slot]} tokens, the table holds {self.max_len}")
        return tokens

    def reserve(self, slots, counts):
        want = {slot: -(-(self.length[slot] + n) // self.page) - self.end[slot] for slot, n in self._tokens(slots, counts).items()}
        if sum(max(w, 0) for w in want.values()) > len(self.free):
            raise RuntimeError(f"the paged cache has {len(self.free)} pages left")
        changed = [slot for slot, w in want.items() if w > 0]
        for slot in changed:
            for _ in range(want[slot]):
                self.table[slot][self.end[slot]] = self.free.pop()
                self.end[slot] += 1
        return changed

    def forget(self, slot, before):
        self._check(slot)
        upto = max(min(before, self.length[slot]), 0) // self.page          # pages of tokens that are yet to come stay
        if upto <= self.first[slot]:
            return []
        row = self.table[slot]
        self.free.extend(row[self.first[slot]:upto])
        row[self.first[slot]:upto] = [-1] * (upto - self.first[slot])
        self.first[slot] = upto
        return [slot]

    def advance(self, slots, counts):
        tokens = self._tokens(slots, counts)
        for slot, n in tokens.items():
            if self.length[slot] + n > self.end[slot] * self.page:
                raise ValueError(f"slot {slot} has no pages for {n} more tokens")
        for slot, n in tokens.items():
            self.length[slot] += n
