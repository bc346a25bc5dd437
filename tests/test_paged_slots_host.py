"""The paged cache's accounts of sequences that end, begin and are refused, on the host alone: the kernels are stood in for by calls that
write nothing."""
import pytest
import torch

from diffcache_amd import PagedCache
from diffcache_amd import _hip as hip


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.fixture
def cache(monkeypatch):
    """A maker of caches on the CPU; what their calls were asked for is in cache.appended and cache.attended."""
    def make(**more):
        return PagedCache(**{**dict(num_layers=2, batch_size=3, max_length=100, num_kv_heads=1, num_q_heads=2, head_dim=64, page_size=16, device="cpu"), **more})

    make.appended, make.attended = [], []

    def append(k_pages, v_pages, table, k, v, start=None, **kw):
        make.appended.append(dict(kw, k=k, table=table.clone(), start=None if start is None else start.tolist(),
                                  counts=None if kw["counts"] is None else kw["counts"].tolist()))
        return kw["q"]

    def attn(q, k_pages, v_pages, table, start, counts=None, out=None, lse=None, **kw):
        make.attended.append(dict(kw, start=start.tolist(), counts=None if counts is None else counts.tolist()))
        out = torch.empty_like(q) if out is None else out
        return out if lse is None else (out, lse)

    monkeypatch.setattr(hip, "paged_append", append)
    monkeypatch.setattr(hip, "paged_attn", attn)
    return make


def prefill(c, seq, lens=None):
    for layer in range(c.num_layers):
        c.prefill_update_kv_cache(bf(c.batch_size, seq, 1, 64), bf(c.batch_size, seq, 1, 64), layer, lens=lens)


def decode(c, layers=None):
    b = c.batch_size
    for layer in range(c.num_layers) if layers is None else layers:
        c.decode_attention(layer, bf(b, 2, 64), bf(b, 1, 1, 64), bf(b, 1, 1, 64))


@pytest.mark.parametrize("page", [64, 16])
def test_no_replay_is_counted_past_max_length(cache, page):
    """100 rows end inside a page of both sizes: a replay behind them would write a row that no token attends to."""
    c = cache(page_size=page)
    prefill(c, 97)
    c.reserve(100)
    c.advance_host_step(2)
    c.advance_host_step()
    assert c.seq_len(0) == 100
    with pytest.raises(AssertionError, match="max_length"):
        c.advance_host_step()
    assert c._lens == [100] * 3
    c.advance_host_step(-1)
    with pytest.raises(AssertionError, match="max_length"):
        c.advance_host_step(2)
    assert c._lens == [99] * 3
