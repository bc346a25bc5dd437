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


def test_a_freed_sequence_is_left_alone_by_decode_steps(cache):
    c = cache(num_pages=14)
    prefill(c, 90, lens=[90, 50, 20])
    c.free(1)
    for step in range(10):
        decode(c)
        assert all(a["counts"] == [1, 0, 1] for a in cache.appended[-2:] + cache.attended[-2:])
        assert c._lens == c.lens.tolist() == [91 + step, 0, 21 + step]
    assert c._pages[1] == [] and (c.table[1] == -1).all() and len(c._free) == 14 - 7 - 2
    with pytest.raises(AssertionError, match="full"):
        decode(c)
    c.free(0)                                                      # (the one that is full)
    decode(c)
    assert c._lens == c.lens.tolist() == [0, 0, 31]
    c.free(2)
    decode(c)                                                      # nothing to do
    assert c._lens == c.lens.tolist() == [0, 0, 0] and sorted(c._free) == list(range(14)) and cache.attended[-1]["counts"] == [0, 0, 0]


def test_a_freed_sequence_does_not_count_in_replays(cache):
    c = cache()
    prefill(c, 40, lens=[40, 33, 8])
    c.free(1)
    c.reserve(60)                                                  # (of the sequences that there are)
    assert [len(p) for p in c._pages] == [4, 0, 4]
    c.advance_host_step(20)
    assert c._lens == [60, 0, 28]
    c.advance_host_step(-3)
    assert c._lens == [57, 0, 25]
    with pytest.raises(AssertionError, match="more steps"):
        c.advance_host_step(8)
    with pytest.raises(AssertionError, match="more steps"):
        c.advance_host_step(-26)
    assert c._lens == [57, 0, 25]


@pytest.mark.parametrize("how", ["extend", "whole extend", "prefill", "share", "share nothing"])
def test_a_freed_sequence_begins_anew(cache, how):
    c = cache()
    prefill(c, 40, lens=[40, 33, 8])
    c.free(1)
    c.reserve([90, 0, 90])                                         # room enough for the others
    decode(c)
    want = [41, 0, 9]
    if how == "extend":
        for layer in range(2):
            c.extend_attention(layer, bf(3, 5, 2, 64), bf(3, 5, 1, 64), bf(3, 5, 1, 64), lens=[0, 5, 0])
            assert len(c._pages[1]) == 1 and (cache.appended[-1]["table"][1] >= 0).sum() == 1
        want = [41, 5, 9]
    elif how == "whole extend":
        for layer in range(2):
            c.extend_attention(layer, bf(3, 20, 2, 64), bf(3, 20, 1, 64), bf(3, 20, 1, 64))
            assert len(c._pages[1]) == 2
        want = [61, 20, 29]
    elif how == "prefill":
        prefill(c, 7, lens=[3, 7, 0])
        want = [3, 7, 0]
    else:
        c.share_prefix(1, 0, 32 if how == "share" else 0)
        want = [41, 32 if how == "share" else 0, 9]
    assert c._lens == c.lens.tolist() == want
    decode(c)
    assert c._lens == c.lens.tolist() == [n + 1 for n in want]
    assert all(len(p) * 16 >= n for n, p in zip(c._lens, c._pages))
    c.reserve(96)
    c.advance_host_step()
    assert c._lens == [n + 2 for n in want]


def test_an_empty_prompt_begins_a_sequence_that_was_not_freed(cache):
    c = cache()
    prefill(c, 7, lens=[7, 0, 3])
    decode(c)
    assert c._lens == c.lens.tolist() == [8, 1, 4]
    c.free(2)
    prefill(c, 5, lens=[5, 0, 0])
    decode(c)
    assert c._lens == c.lens.tolist() == [6, 1, 0]


def test_steps_go_by_what_is_freed_and_filled_when_they_run(cache):
    """One tensor, made with the cache, says which sequences a step counts: a captured step reads it at every replay."""
    c = cache()
    prefill(c, 7)
    live = c.live
    at = live.data_ptr()
    c.free(0)
    c.free(2)
    assert live.tolist() == [0, 1, 0]
    c.share_prefix(2, 1, 0)
    for layer in range(2):
        assert live.tolist() == [0, 1, 1]
        c.extend_attention(layer, bf(3, 2, 2, 64), bf(3, 2, 1, 64), bf(3, 2, 1, 64), lens=[2, 0, 0])
    assert c.live is live and live.tolist() == [1, 1, 1] and live.data_ptr() == at and live.dtype == torch.int32


def state(c):
    return [list(p) for p in c._pages], sorted(c._free), list(c._holders), list(c._lens), list(c._live), c._room, c.table.tolist(), c.lens.tolist(), c.live.tolist()


@pytest.mark.parametrize("layer", [-1, -2, 2, 7])
def test_prompts_for_layers_that_there_are_not_are_refused(cache, layer):
    c = cache()
    for lens in ([40, 33, 8], None):
        before = state(c)
        with pytest.raises(AssertionError, match="no such layer"):
            c.prefill_update_kv_cache(bf(3, 40, 1, 64), bf(3, 40, 1, 64), layer, lens=lens)
        assert state(c) == before and not cache.appended
        c.reserve(20)


@pytest.mark.parametrize("call,refuses", [(call, "append") for call in ("prefill", "padded prefill", "extend", "padded extend", "decode")]
                         + [(call, "attn") for call in ("extend", "padded extend", "decode")])
@pytest.mark.parametrize("shared", [False, True])
def test_a_refused_call_gives_back_the_pages_that_it_took(cache, monkeypatch, call, shared, refuses):
    c = cache()
    prefill(c, 16, lens=[16, 16, 3])
    if shared:
        c.share_prefix(1, 0, 16)
    c.free(2)
    before = state(c)

    def refuse(*a, **kw):
        raise hip.DiffCacheError("k must be bf16")

    calls = {"prefill": lambda: c.prefill_update_kv_cache(bf(3, 50, 1, 64), bf(3, 50, 1, 64), 1),
             "padded prefill": lambda: c.prefill_update_kv_cache(bf(3, 50, 1, 64), bf(3, 50, 1, 64), 1, lens=[50, 0, 20]),
             "extend": lambda: c.extend_attention(1, bf(3, 40, 2, 64), bf(3, 40, 1, 64), bf(3, 40, 1, 64)),
             "padded extend": lambda: c.extend_attention(1, bf(3, 40, 2, 64), bf(3, 40, 1, 64), bf(3, 40, 1, 64), lens=[0, 17, 40]),
             "decode": lambda: decode(c, [1])}
    with monkeypatch.context() as m:
        m.setattr(hip, "paged_" + refuses, refuse)
        for _ in range(2):
            with pytest.raises(hip.DiffCacheError, match="bf16"):
                calls[call]()
            assert state(c) == before
    free = list(c._free)
    calls[call]()                                                  # and goes as if there had been no refused one
    taken = [p for pages, old in zip(c._pages, before[0]) for p in pages if p not in old]
    assert taken and set(taken) <= set(free + sum(before[0], []))
    assert sorted(c._free + list({p for pages in c._pages for p in pages})) == list(range(c.num_pages))


def test_nothing_of_a_freed_sequence_is_handed_out_again(cache):
    """Without `out` a step returns the cache's own tensor: a sequence that is not live has zeros there, not its last outputs."""
    c = cache()
    prefill(c, 7)
    c._attn_out.fill_(3)                                           # (what a step would leave)
    c.free(1)
    got = c.decode_attention(0, bf(3, 2, 64), bf(3, 1, 1, 64), bf(3, 1, 1, 64))
    assert got is c._attn_out and (got[1] == 0).all() and (got[0] == 3).all() and (got[2] == 3).all()


def test_tokens_taken_back_of_all_sequences_leave_a_freed_one_empty(cache):
    c = cache()
    prefill(c, 7)
    c.free(1)
    decode(c)
    c.lens.sub_(1)                                                 # (of the freed one too)
    c.advance_host_step(-1)
    assert c._lens == [7, 0, 7]
    for layer in range(2):
        c.extend_attention(layer, bf(3, 5, 2, 64), bf(3, 5, 1, 64), bf(3, 5, 1, 64), lens=[0, 5, 1])
        assert cache.attended[-1]["start"] == [7, 0, 7]
    assert c._lens == c.lens.tolist() == [7, 5, 8]
    decode(c)
    assert c._lens == c.lens.tolist() == [8, 6, 9]
