"""``MxCache``: a whole context in 4 or 8 bits to a number, every token of it attended to.

``DiffCache`` keeps bf16 rows and attends to a selection of them.  This cache stands beside it for contexts that are
to be attended to as a whole, with the hooks of the reference's cache that such a decoder needs
(``src/diffcache/kvcache/diffcache.py:149-184``, ``src/diffcache/base.py:83,134-142``):

    prefill_update_kv_cache(key_states, value_states, layer_idx)
    decode_attention(layer_idx, queries, key_states, value_states)
    seq_len / seq_len_gpu, advance_host_step

Keys and values are held in blocks of 32 numbers with a power of two (``dc_mx_store`` of the header), 4.25 bits a number with
``key_bits`` / ``value_bits`` 4 and 8.25 with 8: at 4 bits a layer's step reads about what a scan of the 8-bit key
sketch does.  A row is written once, when its token comes, and read as it is held from then on, in its own step too.

The lengths of the sequences live in ``lens``, an int32 tensor on the device (the ``cache_seqlens`` of
``base.py:134-142``): a captured ``decode_attention`` writes to and attends over the rows that it names and counts it
up after the last layer, so a captured step stays right on every replay; ``advance_host_step`` brings the host's mirror
up to date.  Sequences of one batch may have prompts of different lengths.  ``window`` > 0 attends to the first
``sink_len`` and the last ``window`` rows alone.  All layers share one workspace: calls and replays of one cache go one after another
(two caches may run side by side).  A copied or saved cache has memory of its own.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import _hip as hip


class MxCache:
    def __init__(self, num_layers: int, batch_size: int, max_length: int, num_kv_heads: int, num_q_heads: int,
                 head_dim: int, key_bits: int = 4, value_bits: int = 4, sink_len: int = 0, window: int = 0,
                 device: str = "cuda") -> None:
        hip.require(num_layers >= 1 and batch_size >= 1 and max_length >= 1, "a cache needs layers, sequences and rows")
        hip.require(num_kv_heads >= 1 and num_q_heads >= 1 and num_q_heads % num_kv_heads == 0,
                    "num_q_heads must be a multiple of num_kv_heads")
        hip.require(num_q_heads // num_kv_heads <= hip.MX_MAX_GROUP,
                    f"more than {hip.MX_MAX_GROUP} query heads to a KV head are not supported")
        hip.require(sink_len >= 0 and window >= 0, "sink_len and window must not be negative")
        self.num_layers, self.batch_size, self.max_length = num_layers, batch_size, max_length
        self.num_kv_heads, self.num_q_heads, self.head_dim = num_kv_heads, num_q_heads, head_dim
        self.sink_len, self.window = sink_len, window
        self.device = torch.device(device)

        def stores(bits: int):
            return [hip.MxStore.zeros(batch_size, num_kv_heads, max_length, head_dim, bits, self.device)
                    for _ in range(num_layers)]

        self.kstore, self.vstore = stores(key_bits), stores(value_bits)
        self.lens = torch.zeros((batch_size,), dtype=torch.int32, device=self.device)
        self._longest = 0     # the host's mirror of the longest sequence
        self._workspace = torch.empty(
            (hip.mx_attn_workspace_bytes(batch_size * num_kv_heads, num_q_heads // num_kv_heads, head_dim, max_length),),
            dtype=torch.uint8, device=self.device)
        self._attn_out: Optional[torch.Tensor] = None

    def prefill_update_kv_cache(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int,
                                lens: Optional[Sequence[int]] = None):
        """key_states / value_states (bsz, seq_len, num_kv_heads, head_dim) bf16 on the GPU.  ``lens``: the prompts' lengths
        where they are padded to a common one (behind their tokens); the same for every layer."""
        seq = key_states.size(1)
        hip.require(0 < seq <= self.max_length, "the prompt is empty or longer than max_length")
        # a replay would move the rows and leave the host's length as it is
        hip.require(not torch.cuda.is_current_stream_capturing(), "a prefill cannot be captured in a graph")
        at, longest = None, seq
        if lens is not None:
            lens = [int(x) for x in lens]
            hip.require(len(lens) == self.batch_size and all(0 <= x <= seq for x in lens), "lens does not fit the prompts")
            # (from pinned memory: nothing waits for the device)
            at = torch.tensor(lens, dtype=torch.int32, pin_memory=True).to(self.device, non_blocking=True)
            longest = max(lens)
        hip.mx_ingest(self.kstore[layer_idx], self.vstore[layer_idx], key_states, value_states, lens=at)
        # only now: a call that was refused leaves the lengths of what the cache holds
        if at is None:
            self.lens.fill_(seq)
        else:
            self.lens.copy_(at)
        self._longest = longest
        return key_states, value_states

    def decode_attention(self, layer_idx: int, queries: torch.Tensor, key_states: torch.Tensor,
                         value_states: torch.Tensor, out: Optional[torch.Tensor] = None,
                         lse: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One layer of a decode step: write the token's k/v behind each sequence and attend to all of it (or to its sinks and
        window).  queries (bsz, 1, Hq*hd) or (bsz, Hq, hd); key/value_states (bsz, 1, Hkv, hd).  Returns (bsz, Hq, hd)
        bf16; ``lse`` (bsz, Hq) fp32 receives the log of the sum of exponentials.  Call it for every layer of a step; the
        sequences grow by one after the last layer."""
        b, hq, hd = self.batch_size, self.num_q_heads, self.head_dim
        capturing = torch.cuda.is_current_stream_capturing()
        hip.require(self._longest < self.max_length, "the cache is full (max_length)")
        if out is None:
            if self._attn_out is None:
                self._attn_out = torch.empty((b, hq, hd), device=self.device, dtype=torch.bfloat16)
            out = self._attn_out
        # a captured launch is laid out for the longest sequences that the cache holds, and goes by lens when it runs
        hip.mx_attn(queries.reshape(b, hq, hd), self.kstore[layer_idx], self.vstore[layer_idx], self.lens,
                    n_rows=self.max_length if capturing else self._longest + 1, n_sink=self.sink_len,
                    window=self.window, new_k=key_states, new_v=value_states, out=out, lse=lse,
                    workspace=self._workspace)
        if layer_idx == self.num_layers - 1:
            self.lens.add_(1)
            if not capturing:   # a captured step is counted when it is replayed (advance_host_step)
                self._longest += 1
        return out

    def advance_host_step(self, steps: int = 1) -> None:
        """After ``steps`` replays of a captured decode step: bring the host's mirror of the longest sequence up to the
        device's lengths (no synchronisation).  Negative: tokens taken back, which ``lens.sub_`` takes off the device's."""
        hip.require(0 <= self._longest + steps <= self.max_length, "more steps were replayed than the cache has rows")
        self._longest += steps

    def get_kvcache(self, layer_idx: int):
        """K and V of a layer as bf16 (bsz, kv_heads, seq_len, head_dim); rows behind a shorter sequence's end are whatever
        the store holds there (zeros where nothing was written)."""
        return hip.mx_gather_rows(self.kstore[layer_idx], self.vstore[layer_idx], n_idx=self._longest)

    def seq_len(self, layer_idx: int) -> int:
        return self._longest

    def seq_len_gpu(self, layer_idx: int) -> int:
        return self._longest
