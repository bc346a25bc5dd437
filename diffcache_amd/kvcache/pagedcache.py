"""``PagedCache``: bf16 keys and values in pages, every token of a sequence attended to.

``DiffCache`` and ``MxCache`` reserve ``max_length`` rows for every sequence.  This cache stands beside them for batches whose
sequences differ in length, grow, or begin alike: a layer has a pool of pages of ``page_size`` rows, a sequence holds those that its
rows need, and two sequences may hold the pages of a common beginning together.  It has the hooks of the reference's cache that
a decoder needs (``src/diffcache/kvcache/diffcache.py:149-184``, ``src/diffcache/base.py:83,134-142``), and one for several
tokens at a time:

    prefill_update_kv_cache(key_states, value_states, layer_idx)
    extend_attention(layer_idx, queries, key_states, value_states)    a prompt's next tokens, or drafted ones
    decode_attention(layer_idx, queries, key_states, value_states)
    seq_len / seq_len_gpu, advance_host_step
    reserve, share_prefix, free

With ``inv_freq`` the cache rotates keys and queries by their positions on their way (``base.py:121-125``), so a model hands them over as its
projections leave them.

``lens`` (int32, on the device) holds the lengths of the sequences and ``table`` their pages, the same for all layers.  A captured
``decode_attention`` goes by both when it is replayed; pages are handed out on the host, so ``reserve`` has to give the sequences
room for the replays first.  A sequence that was given up (``free``) holds nothing and takes no part in decode steps, captured ones
among them, until a prompt or a shared beginning takes its place: ``live`` (int32, on the device) is 0 for it, else 1.  All layers share one
workspace: calls and replays of one cache go one after another (two caches may run side by side).
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from .. import _hip as hip


class PagedCache:
    def __init__(self, num_layers: int, batch_size: int, max_length: int, num_kv_heads: int, num_q_heads: int,
                 head_dim: int, page_size: int = 64, num_pages: Optional[int] = None, sink_len: int = 0, window: int = 0,
                 inv_freq: Optional[torch.Tensor] = None, interleaved: bool = False,
                 sections: Optional[Tuple[int, ...]] = None, device: str = "cuda") -> None:
        hip.require(num_layers >= 1 and batch_size >= 1 and max_length >= 1, "a cache needs layers, sequences and rows")
        hip.require(num_kv_heads >= 1 and num_q_heads >= 1 and num_q_heads % num_kv_heads == 0,
                    "num_q_heads must be a multiple of num_kv_heads")
        hip.require(num_q_heads // num_kv_heads <= hip.PAGED_MAX_GROUP,
                    f"more than {hip.PAGED_MAX_GROUP} query heads to a KV head are not supported")
        hip.require(head_dim in (64, 128, 256), f"head_dim {head_dim} is not supported (64, 128 or 256)")
        hip.require(16 <= page_size <= 65536 and page_size & (page_size - 1) == 0, "page_size must be a power of two from 16 to 65536")
        hip.require(sink_len >= 0 and window >= 0, "sink_len and window must not be negative")
        hip.require(sections is None or inv_freq is not None, "sections are of a rotation: inv_freq is missing")
        self.num_layers, self.batch_size, self.max_length = num_layers, batch_size, max_length
        self.num_kv_heads, self.num_q_heads, self.head_dim, self.page_size = num_kv_heads, num_q_heads, head_dim, page_size
        self.sink_len, self.window = sink_len, window
        self.device = torch.device(device)
        wide = (max_length + page_size - 1) // page_size
        self.num_pages = batch_size * wide if num_pages is None else num_pages
        hip.require(self.num_pages >= 1, "a cache needs a page")

        def pools():
            return [torch.zeros((self.num_pages, num_kv_heads, page_size, head_dim), dtype=torch.bfloat16, device=self.device)
                    for _ in range(num_layers)]

        self.k_pages, self.v_pages = pools(), pools()
        self.inv_freq = None if inv_freq is None else inv_freq.to(device=self.device, dtype=torch.float32).contiguous()
        self.interleaved, self.sections = interleaved, sections
        self.lens = torch.zeros((batch_size,), dtype=torch.int32, device=self.device)
        self.table = torch.full((batch_size, wide), -1, dtype=torch.int32, device=self.device)
        self.live = torch.ones((batch_size,), dtype=torch.int32, device=self.device)
        self._lens: List[int] = [0] * batch_size                     # the host's mirror of lens
        self._live: List[int] = [1] * batch_size                     # and of live
        self._pages: List[List[int]] = [[] for _ in range(batch_size)]
        self._free = list(range(self.num_pages - 1, -1, -1))
        self._holders = [0] * self.num_pages                         # sequences that hold a page
        self._room = 0                                               # tokens that every live sequence has pages for
        self._workspace = torch.empty(
            (hip.paged_attn_workspace_bytes(batch_size, num_kv_heads, num_q_heads // num_kv_heads, head_dim, max_length),),
            dtype=torch.uint8, device=self.device)
        # (made here: one that a captured step made would be the graph's; zeros, for what stays there of sequences that are not live)
        self._attn_out = torch.zeros((batch_size, num_q_heads, head_dim), device=self.device, dtype=torch.bfloat16)
        self._q = torch.empty_like(self._attn_out) if self.rotates else None

    @property
    def rotates(self) -> bool:
        """Whether keys and queries are handed over as the projections leave them."""
        return self.inv_freq is not None

    # ---- pages, on the host ----

    def reserve(self, lengths: Union[int, Sequence[int]]) -> None:
        """Pages for rows 0 .. lengths[i] - 1 of every sequence (an int: of each of them that is live).  A call that the pool has too
        few pages for changes nothing."""
        self._reserve([lengths * x for x in self._live] if isinstance(lengths, int) else [int(n) for n in lengths])

    def _reserve(self, lengths: Sequence[int]) -> List[int]:
        """The pages that every sequence got, for _take_back."""
        hip.require(len(lengths) == self.batch_size and all(0 <= n <= self.max_length for n in lengths),
                    "lengths must be one for every sequence, up to max_length")
        need = [max((n + self.page_size - 1) // self.page_size - len(p), 0) for n, p in zip(lengths, self._pages)]
        self._hand_out(need, [])
        return need

    def _hand_out(self, need: Sequence[int], dropped: Sequence[int]) -> None:
        """need[i] more pages for sequence i, after the sequences in ``dropped`` gave theirs back."""
        freed = sum(1 for p in self._held_by(dropped))
        hip.require(sum(need) <= len(self._free) + freed, f"the cache has too few pages left ({len(self._free)} of {self.num_pages})")
        if not any(need) and not dropped:
            return
        # a replay would not hand out pages again
        hip.require(not self._capturing(), "pages cannot be handed out while a graph is captured: reserve them before")
        for i in dropped:
            self._give_back(i)
        for pages, n in zip(self._pages, need):
            for _ in range(n):
                page = self._free.pop()
                self._holders[page] = 1
                pages.append(page)
        self._upload()

    def _take_back(self, need: Sequence[int]) -> None:
        """The last need[i] pages of every sequence, as they were before _hand_out."""
        if not any(need):
            return
        for pages, n in reversed(list(zip(self._pages, need))):
            for _ in range(n):
                page = pages.pop()
                self._holders[page] = 0
                self._free.append(page)
        self._upload()

    def _held_by(self, sequences: Sequence[int]) -> List[int]:
        """Pages that no one would hold without these sequences."""
        left = {}
        for i in sequences:
            for p in self._pages[i]:
                left[p] = left.get(p, self._holders[p]) - 1
        return [p for p, n in left.items() if n == 0]

    def _give_back(self, i: int) -> None:
        for p in self._pages[i]:
            self._holders[p] -= 1
            if self._holders[p] == 0:
                self._free.append(p)
        self._pages[i] = []

    def _upload(self) -> None:
        wide = self.table.shape[1]
        rows = [p + [-1] * (wide - len(p)) for p in self._pages]
        # (from pinned memory: nothing waits for the device)
        self.table.copy_(self._pinned(rows), non_blocking=True)
        self._count_room()

    def _pinned(self, numbers) -> torch.Tensor:
        return torch.tensor(numbers, dtype=torch.int32, pin_memory=self.device.type == "cuda")

    def _count_room(self) -> None:
        self._room = min((len(p) * self.page_size - n for p, n, x in zip(self._pages, self._lens, self._live) if x), default=0)

    def _set_live(self, live: Sequence[int]) -> None:
        if list(live) != self._live:
            self._live = list(live)
            self.live.copy_(self._pinned(self._live), non_blocking=True)

    def _with(self, counts: Sequence[int]) -> List[int]:
        """live, with the sequences that these tokens are of."""
        return [1 if n else x for n, x in zip(counts, self._live)]

    @staticmethod
    def _capturing() -> bool:
        return torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()

    def share_prefix(self, sequence: int, of: int, rows: int) -> None:
        """Sequence ``sequence`` begins anew with the first ``rows`` rows of sequence ``of``, whose pages both hold from then on; ``rows`` is
        a multiple of page_size that ``of`` holds in all layers.  No row of these pages is written any more: both go on behind them."""
        hip.require(0 <= sequence < self.batch_size and 0 <= of < self.batch_size and sequence != of, "no such sequences")
        hip.require(0 <= rows <= self._lens[of] and rows % self.page_size == 0, "rows must be whole pages of the other sequence")
        hip.require(not self._capturing(), "pages cannot be handed out while a graph is captured")
        pages = self._pages[of][:rows // self.page_size]
        for p in pages:
            self._holders[p] += 1
        self._give_back(sequence)
        self._pages[sequence] = list(pages)
        self._lens[sequence] = rows
        self.lens[sequence:sequence + 1].fill_(rows)
        self._set_live([1 if i == sequence else x for i, x in enumerate(self._live)])
        self._upload()

    def free(self, sequence: int) -> None:
        """Sequence ``sequence`` holds nothing any more; its pages are others' to take.  Decode steps leave it alone until
        ``extend_attention`` or ``prefill_update_kv_cache`` has tokens of it or ``share_prefix`` begins it anew."""
        hip.require(0 <= sequence < self.batch_size, "no such sequence")
        hip.require(not self._capturing(), "pages cannot be given back while a graph is captured")
        self._give_back(sequence)
        self._lens[sequence] = 0
        self.lens[sequence:sequence + 1].zero_()
        self._attn_out[sequence].zero_()        # (no step writes it until the sequence begins anew)
        self._set_live([0 if i == sequence else x for i, x in enumerate(self._live)])
        self._upload()

    # ---- the decoder's hooks ----

    def _append(self, layer_idx: int, k: torch.Tensor, v: torch.Tensor, start: Optional[torch.Tensor], counts: Optional[torch.Tensor],
                q: Optional[torch.Tensor], q_out: Optional[torch.Tensor], pos: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
        return hip.paged_append(self.k_pages[layer_idx], self.v_pages[layer_idx], self.table, k, v, start, counts=counts, q=q, q_out=q_out,
                                inv_freq=self.inv_freq, interleaved=self.interleaved, pos=pos, sections=self.sections)

    def _counts(self, lens: Optional[Sequence[int]], most: int):
        """(lengths on the host, the same on the device or None) of tokens that may be padded."""
        if lens is None:
            return [most] * self.batch_size, None
        lens = [int(x) for x in lens]
        hip.require(len(lens) == self.batch_size and all(0 <= x <= most for x in lens), "lens does not fit the tokens")
        return lens, self._pinned(lens).to(self.device, non_blocking=True)

    def prefill_update_kv_cache(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
                                lens: Optional[Sequence[int]] = None, pos: Optional[torch.Tensor] = None):
        """key_states / value_states (bsz, seq_len, num_kv_heads, head_dim) bf16 on the GPU take the place of what the sequences held.
        ``lens``: the prompts' lengths where they are padded to a common one (behind their tokens); the same for every layer.  ``pos``: positions
        of the tokens, (bsz, seq_len) int32, or (bsz, seq_len, axes) with sections; their rows without it."""
        seq = key_states.size(1)
        hip.require(0 <= layer_idx < self.num_layers, "no such layer")
        hip.require(0 < seq <= self.max_length, "the prompt is empty or longer than max_length")
        # a replay would move the rows and leave the host's lengths as they are
        hip.require(not self._capturing(), "a prefill cannot be captured in a graph")
        at, counts = self._counts(lens, seq)
        self._check_states(key_states, value_states, (self.batch_size, seq))
        # pages that others hold too stay theirs
        dropped = [i for i, p in enumerate(self._pages) if any(self._holders[x] > 1 for x in p)]
        need = [max((n + self.page_size - 1) // self.page_size - (0 if i in dropped else len(self._pages[i])), 0) for i, n in enumerate(at)]
        before = ([list(p) for p in self._pages], list(self._holders), list(self._free)) if dropped else None
        self._hand_out(need, dropped)
        try:
            self._append(layer_idx, key_states, value_states, None, counts, None, None, pos)
        except Exception:
            if before is None:
                self._take_back(need)
            else:          # the pages that were given back hold rows yet
                self._pages, self._holders, self._free = before
                self._upload()
            raise
        # only now: a call that was refused leaves the lengths of what the cache holds
        if counts is None:
            self.lens.fill_(seq)
        else:
            self.lens.copy_(counts)
        self._lens = at
        self._set_live(self._with(at))
        self._count_room()
        return key_states, value_states

    def _check_states(self, k: torch.Tensor, v: torch.Tensor, lead) -> None:
        want = (*lead, self.num_kv_heads, self.head_dim)
        hip.require(tuple(k.shape) == want and tuple(v.shape) == want, f"key_states and value_states must be {want}")

    def _attend(self, layer_idx: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, at: List[int], counts: Optional[torch.Tensor],
                out: Optional[torch.Tensor], lse: Optional[torch.Tensor], pos: Optional[torch.Tensor], workspace, q_out) -> torch.Tensor:
        hip.require(0 <= layer_idx < self.num_layers, "no such layer")
        capturing = self._capturing()
        grown = [n + c for n, c in zip(self._lens, at)]
        hip.require(max(grown) <= self.max_length, "the cache is full (max_length)")
        live = at if at is self._live else self._with(at)       # (a decode step has one token of each)
        need = self._reserve(grown) if max(at) > self._room or live != self._live else []
        if live != self._live:
            for i, (x, y) in enumerate(zip(live, self._live)):
                if x > y:   # (tokens that were taken back of all sequences may have gone off a freed one's too)
                    self.lens[i:i + 1].zero_()
        try:
            turned = self._append(layer_idx, k, v, self.lens, counts, q if self.rotates else None, q_out, pos)
            got = hip.paged_attn(q if turned is None else turned, self.k_pages[layer_idx], self.v_pages[layer_idx], self.table, self.lens,
                                 counts=counts,
                                 # a captured launch is laid out for the longest sequences that the cache holds, and goes by lens when it runs
                                 n_rows=self.max_length if capturing else max(max(grown), 1),
                                 n_sink=self.sink_len, window=self.window, out=out, lse=lse, workspace=workspace)
        except Exception:
            self._take_back(need)
            raise
        if layer_idx == self.num_layers - 1:
            self.lens.add_(q.shape[1] if q.dim() == 4 else 1) if counts is None else self.lens.add_(counts)
            if not capturing:   # a captured step is counted when it is replayed (advance_host_step)
                self._lens = grown
                self._set_live(live)
                self._count_room()
        return got if lse is None else got[0]

    def extend_attention(self, layer_idx: int, queries: torch.Tensor, key_states: torch.Tensor, value_states: torch.Tensor,
                         lens: Optional[Sequence[int]] = None, out: Optional[torch.Tensor] = None,
                         lse: Optional[torch.Tensor] = None, pos: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One layer of a step of several tokens: write their k/v behind each sequence and attend, every token up to its own row.
        queries (bsz, tokens, Hq, hd), key/value_states (bsz, tokens, Hkv, hd); ``lens``: the tokens that a sequence has of them, the
        same for every layer.  Returns (bsz, tokens, Hq, hd) bf16, of which padded tokens' stay what ``out`` held; ``lse`` (bsz, tokens,
        Hq) fp32 receives the log of the sum of exponentials.  Call it for every layer; the sequences grow after the last one."""
        # (a replay would not hand out pages, nor know the lengths)
        hip.require(not self._capturing(), "only a decode step can be captured in a graph")
        hip.require(queries.dim() == 4 and tuple(queries.shape[2:]) == (self.num_q_heads, self.head_dim) and queries.size(0) == self.batch_size
                    and queries.size(1) > 0, f"queries must be (bsz, tokens, {self.num_q_heads}, {self.head_dim})")
        self._check_states(key_states, value_states, tuple(queries.shape[:2]))
        at, counts = self._counts(lens, queries.size(1))
        return self._attend(layer_idx, queries, key_states, value_states, at, counts, out, lse, pos, None, None)

    def decode_attention(self, layer_idx: int, queries: torch.Tensor, key_states: torch.Tensor, value_states: torch.Tensor,
                         out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                         pos: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One layer of a decode step: write the token's k/v behind each sequence and attend to all of it (or to its sinks and
        window).  queries (bsz, 1, Hq*hd) or (bsz, Hq, hd); key/value_states (bsz, 1, Hkv, hd); ``pos`` (bsz) int32, or (bsz, axes).  Returns
        (bsz, Hq, hd) bf16, ``out`` or a tensor of the cache's that the next call writes again; ``lse`` (bsz, Hq) fp32 receives the log of the sum of exponentials.  Call it for every layer of a step; the
        sequences grow by one after the last layer.  Those that are not live are left alone: their rows of ``out`` and ``lse`` stay what they were (those of the
        cache's own tensor are zeros)."""
        b, hq, h, hd = self.batch_size, self.num_q_heads, self.num_kv_heads, self.head_dim
        if out is None:
            out = self._attn_out
        return self._attend(layer_idx, queries.reshape(b, hq, hd), key_states.reshape(b, h, hd), value_states.reshape(b, h, hd),
                            self._live, self.live, out, lse, pos, self._workspace, self._q)

    def advance_host_step(self, steps: int = 1) -> None:
        """After ``steps`` replays of a captured decode step: bring the host's mirror of the lengths up to the device's (no
        synchronisation).  Negative: tokens taken back of the live sequences, which ``lens.sub_`` takes off the device's."""
        grown = [n + steps * x for n, x in zip(self._lens, self._live)]
        # (a step is captured for max_length rows: of one behind them in the last page a token would be written and never attended to)
        hip.require(min(grown) >= 0 and max(grown) <= self.max_length and all(n <= len(p) * self.page_size for n, p in zip(grown, self._pages)),
                    "more steps were replayed than the sequences have pages, or rows up to max_length")
        hip.require(all(n >= self.page_size * sum(1 for x in p if self._holders[x] > 1) for n, p in zip(grown, self._pages)),
                    "rows of pages that two sequences hold cannot be taken back")
        self._lens = grown
        self._count_room()

    def get_kvcache(self, layer_idx: int):
        """K and V of a layer as bf16 (bsz, kv_heads, seq_len, head_dim); rows behind a shorter sequence's end hold anything."""
        n = max(self._lens)
        at = self.table.long().clamp(min=0)

        def rows(pool: torch.Tensor) -> torch.Tensor:
            return pool[at].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n].contiguous()

        return rows(self.k_pages[layer_idx]), rows(self.v_pages[layer_idx])

    def seq_len(self, layer_idx: int) -> int:
        return max(self._lens)

    def seq_len_gpu(self, layer_idx: int) -> int:
        return max(self._lens)
