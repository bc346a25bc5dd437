"""The paged cache without a GPU: struct layouts, every refusal, the pages' accounts, and the plain form's own properties."""
import ctypes
import math
import os
import re

import pytest
import torch

from diffcache_amd import PagedCache
from diffcache_amd import _hip as hip
from oracle import paged as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 22   # an address that no kernel is launched on: every call below is refused first


@pytest.mark.parametrize("name,cls", [("dc_paged_store", hip.PagedStoreArgs), ("dc_paged_tokens", hip.PagedTokensArgs),
                                      ("dc_paged_append_args", hip.PagedAppendArgs), ("dc_paged_attn_args", hip.PagedAttnArgs)])
def test_structs_match_the_header(name, cls):
    header = open(os.path.join(ROOT, "include", "diffcache_hip.h")).read()
    body = header[header.index("typedef struct %s {" % name):header.index("} %s;" % name)]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    names = [re.sub(r"\[.*|[^A-Za-z0-9_]", "", n.split()[-1]) for decl in body.split(";") if decl.strip()
             for n in decl.replace("*", " ").split(",")]
    assert names == [n for n, _ in cls._fields_]


def store(**change):
    s = hip.PagedStoreArgs(P, 2 * P, 2 * 64 * 128, 64 * 128, 2 * 64 * 128, 64 * 128, 8, 64)
    for n, x in change.items():
        setattr(s, n, x)
    return s


def tokens(**change):
    t = hip.PagedTokensArgs(P, P, None, None, 8, 2, 4, 8, 8)
    for n, x in change.items():
        setattr(t, n, x)
    return t


def append_args(**change):
    a = hip.PagedAppendArgs(P, P, P, P, P, None, store(), tokens(), *[1024] * 9, 2, 8, 128, 128, 0, 1, (ctypes.c_int * 4)())
    for n, x in change.items():
        setattr(a, n, x)
    return a


def attn_args(**change):
    a = hip.PagedAttnArgs(P, P, None, store(), tokens(), 1024, 1024, 128, P, 1 << 30, 2, 4, 128, 512, 0, 0, 0.1)
    for n, x in change.items():
        setattr(a, n, x)
    return a


def refused(rc, message, code=-22):
    assert rc == code and re.search(message, hip.lib.dc_last_error().decode()), (rc, hip.lib.dc_last_error())


def test_packed_bytes_are_the_structs():
    s, t = list(range(1, 9)), list(range(11, 20))
    sec = (ctypes.c_int * 4)(61, 62, 63, 64)
    packed = hip._PAGED_APPEND.pack(*range(21, 27), *s, *t, *range(31, 40), *range(41, 47), *sec)
    want = hip.PagedAppendArgs(*range(21, 27), hip.PagedStoreArgs(*s), hip.PagedTokensArgs(*t), *range(31, 40), *range(41, 47), sec)
    assert packed == bytes(want)
    packed = hip._PAGED_ATTN.pack(21, 22, 23, *s, *t, *range(31, 34), 35, 36, *range(41, 47), 0.25)
    assert packed == bytes(hip.PagedAttnArgs(21, 22, 23, hip.PagedStoreArgs(*s), hip.PagedTokensArgs(*t), *range(31, 34), 35, 36, *range(41, 47), 0.25))


BAD = [
    (dict(store=store(k=None)), "null"), (dict(store=store(v=None)), "null"), (dict(store=store(k=P + 8)), "aligned"), (dict(store=store(page=48)), "power of two"),
    (dict(store=store(page=8)), "power of two"), (dict(store=store(page=1 << 17)), "power of two"), (dict(store=store(n_pages=0)), "needs a page"),
    (dict(store=store(v_head_stride=4)), "multiples of 8"), (dict(store=store(k_page_stride=-64)), "negative"), (dict(tokens=tokens(table=None)), "bad table"),
    (dict(tokens=tokens(table_pages=0)), "bad table"), (dict(tokens=tokens(table_stride=7)), "bad table"), (dict(tokens=tokens(cu=P, counts=P)), "different ways"),
    (dict(tokens=tokens(table_pages=1 << 25, table_stride=1 << 25)), "2\\^30"), (dict(tokens=tokens(n_b=-1)), "bad sizes"), (dict(tokens=tokens(max_new=-1)), "bad sizes"),
    (dict(tokens=tokens(n_tokens=-1)), "bad sizes"), (dict(tokens=tokens(max_new=1 << 30)), "too many tokens"), (dict(tokens=tokens(n_b=1 << 23)), "too many units"),
    (dict(n_h=0), "bad sizes"), (dict(hd=96), "head_dim"),
]


@pytest.mark.parametrize("change,message", BAD)
def test_bad_pages_and_tokens_are_refused_everywhere(change, message):
    refused(hip.lib.dc_paged_append_bf16(bytes(append_args(**change)), None), message)
    refused(hip.lib.dc_paged_attn_bf16(bytes(attn_args(**change)), None), message)


@pytest.mark.parametrize("change,message", [
    (dict(k_src=None), "null"), (dict(v_src=None), "null"), (dict(q_src=None), "both"), (dict(q_out=None), "both"), (dict(q_src=None, q_out=None), "n_q"), (dict(n_q=0), "n_q"),
    (dict(k_src=P + 2), "aligned"), (dict(q_out=P + 8), "aligned"), (dict(v_token_stride=12), "multiples of 8"), (dict(q_head_stride=4), "multiples of 8"),
    (dict(rot=24), "rotated"), (dict(rot=144), "rotated"), (dict(rot=-16), "rotated"), (dict(inv_freq=None), "null"), (dict(rot=0), "nothing is rotated"),
    (dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"), (dict(n_axes=2), "positions"), (dict(n_axes=3, pos=P, section=(ctypes.c_int * 4)(16, 24, 23)), "hold 63"),
    (dict(n_axes=2, pos=P, section=(ctypes.c_int * 4)(-1, 65)), "bad section"), (dict(store=store(k_page_stride=0)), "share"), (dict(store=store(v_head_stride=0)), "share"),
    (dict(store=store(k_head_stride=64 * 128 - 8)), "share"),
])
def test_bad_appends_are_refused(change, message):
    refused(hip.lib.dc_paged_append_bf16(bytes(append_args(**change)), None), message)


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(q=P + 8), "aligned"), (dict(out=P + 8), "aligned"), (dict(q_token_stride=4), "multiples of 8"), (dict(group=0), "group"),
    (dict(group=17), "group"), (dict(n_rows=0), "outside"), (dict(n_rows=513), "outside"), (dict(n_sink=-1), "negative"), (dict(window=-1), "negative"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(tokens=tokens(table_pages=4096, table_stride=4096), n_rows=1 << 18, workspace=None), "workspace"),
    (dict(tokens=tokens(table_pages=4096, table_stride=4096), n_rows=1 << 18, workspace=P + 16), "workspace"),
])
def test_bad_attention_is_refused(change, message):
    refused(hip.lib.dc_paged_attn_bf16(bytes(attn_args(**change)), None), message)


def test_a_small_workspace_is_refused():
    a = attn_args(tokens=tokens(table_pages=4096, table_stride=4096), n_rows=1 << 18, workspace_bytes=4096)
    refused(hip.lib.dc_paged_attn_bf16(bytes(a), None), "needed", -12)
    refused(hip.lib.dc_paged_attn_bf16(None, None), "null")
    refused(hip.lib.dc_paged_append_bf16(None, None), "null")


def test_nothing_to_do_is_no_error():
    for t in (tokens(n_b=0), tokens(max_new=0)):
        assert hip.lib.dc_paged_append_bf16(bytes(append_args(tokens=t, k_src=None)), None) == 0
        assert hip.lib.dc_paged_attn_bf16(bytes(attn_args(tokens=t, q=None)), None) == 0


def test_enough_workspace_for_more_is_enough_for_fewer():
    rows = (0, 1, 64, 65, 1000, 100000, 2**30)
    for hd in (64, 128, 256):
        for group in (1, 4, 16):
            for new in range(1, 16 // group + 1):
                for h in (1, 3, 8, 2000):
                    last = [0] * len(rows)
                    for b in (1, 2, 7, 64, 65, 192, 193, 300, 512, 513, 5000):
                        sizes = [hip.paged_attn_workspace_bytes(b, h, group, hd, n, new) for n in rows]
                        assert sizes == sorted(sizes) and all(x >= y for x, y in zip(sizes, last)), (b, h, sizes)
                        last = sizes
                        if new > 1:
                            assert all(x >= y for x, y in zip(sizes, [hip.paged_attn_workspace_bytes(b, h, group, hd, n, new - 1) for n in rows]))
    assert hip.paged_attn_workspace_bytes(0, 1, 4, 128, 100) == hip.paged_attn_workspace_bytes(4, 1, 17, 128, 100) == 0
    assert hip.paged_attn_workspace_bytes(4, 1, 4, 128, -1) == hip.paged_attn_workspace_bytes(4, 1, 4, 128, 100, 0) == 0
    assert hip.paged_attn_workspace_bytes(1 << 20, 1 << 5, 4, 128, 1 << 20) == 0


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def test_wrappers_refuse_what_does_not_fit(monkeypatch):
    monkeypatch.setattr(hip, "_mx_dev", lambda t, name: t.data_ptr())       # so that the checks behind the first tensor's place are reached
    monkeypatch.setattr(hip, "_device", lambda: -1)
    pool, table = bf(4, 2, 16, 64), i32(3, 5)
    k, q = bf(3, 2, 64), bf(3, 4, 64)
    bad = pytest.raises(hip.DiffCacheError)

    def no(message, call):
        with bad as e:
            call()
        assert re.search(message, str(e.value)), e.value

    append = lambda *a, **kw: lambda: hip.paged_append(*a, **kw)  # noqa: E731
    attn = lambda *a, **kw: lambda: hip.paged_attn(*a, **kw)  # noqa: E731
    no("one shape", append(pool, bf(4, 2, 32, 64), table, k, k))
    no("one shape", append(pool.float(), pool.float(), table, k, k))
    no("one after another", append(pool.transpose(1, 2), pool.transpose(1, 2), table, bf(3, 16, 64), bf(3, 16, 64)))
    no("head_dim 32", append(bf(4, 2, 16, 32), bf(4, 2, 16, 32), table, bf(3, 2, 32), bf(3, 2, 32)))
    no("head_dim 4", attn(bf(3, 4, 4), bf(4, 2, 16, 4), bf(4, 2, 16, 4), table))
    no("needs a page", append(pool[:0], pool[:0], table, k, k))
    no("int32 tensor", append(pool, pool, table.long(), k, k))
    no("int32 tensor", append(pool, pool, table[0], k, k))
    no("contiguous rows", append(pool, pool, i32(5, 3).t(), k, k))
    no("k must be", append(pool, pool, table, bf(2, 2, 64), bf(2, 2, 64)))
    no("k must be", append(pool, pool, table, bf(3, 1, 1, 2, 64), k))
    no("k must be bf16", append(pool, pool, table, bf(3, 2, 32), bf(3, 2, 32)))
    no("v must be bf16", append(pool, pool, table, k, bf(3, 3, 64)))
    no("packed", append(pool, pool, table, bf(3, 1, 2, 64), bf(3, 1, 2, 64), cu=i32(4)))
    no("counts are not given", append(pool, pool, table, k, k, cu=i32(4), counts=i32(3)))
    no("cu must be", append(pool, pool, table, k, k, cu=i32(3)))
    no("max_new is 2", append(pool, pool, table, k, k, max_new=2))
    no("start must be", append(pool, pool, table, k, k, i32(2)))
    no("start must be", append(pool, pool, table, k, k, i32(3).long()))
    no("inv_freq is missing", append(pool, pool, table, k, k, q=q))
    no("inv_freq must be", append(pool, pool, table, k, k, inv_freq=torch.zeros(32, dtype=torch.float64)))
    no("need pos", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), sections=(16, 16)))
    no("one to four", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), sections=(), pos=i32(3, 0)))
    no("pos must be", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), pos=i32(3, 2)))
    no("pos must be", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), sections=(16, 16), pos=i32(3)))
    no("q must be bf16", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), q=bf(2, 4, 64)))
    no("q_out must be", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), q=q, q_out=bf(3, 4, 32)))
    no("without q", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), q_out=q))
    no("does not fit its type", append(pool, pool, table, k, k, inv_freq=torch.zeros(32), sections=(1 << 40, 16), pos=i32(3, 2)))
    no("4 heads of 64 numbers, the store 3", attn(q, bf(4, 3, 16, 64), bf(4, 3, 16, 64), table))
    no("more than 16", attn(bf(3, 34, 64), pool, pool, table))
    no("outside the table", attn(q, pool, pool, table, n_rows=81))
    no("outside the table", attn(q, pool, pool, table, n_rows=0))
    no("out must be", attn(q, pool, pool, table, out=bf(3, 3, 64)))
    no("lse must be", attn(q, pool, pool, table, lse=torch.zeros(3, 5)))
    no("workspace must be", attn(q, pool, pool, table, workspace=torch.zeros(8, 8).t()))
    no("does not fit its type", attn(q, pool, pool, table, window=1 << 40))
    monkeypatch.setattr(hip, "_stream", lambda: 0)
    no("scale", attn(q, pool, pool, table, scale=-1.0))
    monkeypatch.undo()
    no("GPU memory", append(pool, pool, table, k, k))


# ---- the cache's pages ----------------------------------------------------------------------------------------------

def cache(**more):
    return PagedCache(**{**dict(num_layers=1, batch_size=3, max_length=100, num_kv_heads=1, num_q_heads=2, head_dim=64, page_size=16, device="cpu"), **more})


def test_pages_are_handed_out_and_given_back():
    c = cache(num_pages=10)
    assert c.table.shape == (3, 7) and c.num_pages == 10
    c.reserve([20, 0, 1])
    assert [len(p) for p in c._pages] == [2, 0, 1] and len(c._free) == 7
    assert c.table[0, :2].tolist() == c._pages[0] and (c.table[0, 2:] == -1).all() and (c.table[1] == -1).all()
    c.reserve([17, 5, 16])                               # what there is already is not handed out again
    assert [len(p) for p in c._pages] == [2, 1, 1]
    before = c.table.clone()
    with pytest.raises(AssertionError, match="too few pages"):
        c.reserve(100)
    assert torch.equal(c.table, before) and len(c._free) == 6
    with pytest.raises(AssertionError, match="max_length"):
        c.reserve(101)
    with pytest.raises(AssertionError, match="max_length"):
        c.reserve([1, 2])
    c.free(0)
    assert len(c._free) == 8 and (c.table[0] == -1).all()
    assert len(set(c._free) | set(c._pages[1]) | set(c._pages[2])) == 10


def test_a_shared_prefix_is_held_until_the_last_one_lets_go():
    c = cache(num_pages=10)
    c.reserve([48, 0, 0])
    c._lens[0] = 40
    with pytest.raises(AssertionError, match="whole pages"):
        c.share_prefix(1, 0, 20)
    with pytest.raises(AssertionError, match="whole pages"):
        c.share_prefix(1, 0, 48)
    with pytest.raises(AssertionError, match="no such"):
        c.share_prefix(0, 0, 16)
    c.share_prefix(1, 0, 32)
    c.share_prefix(2, 1, 16)
    assert c.lens.tolist()[1:] == [32, 16] and c._pages[1] == c._pages[0][:2] and c._pages[2] == c._pages[0][:1]
    assert [c._holders[p] for p in c._pages[0]] == [3, 2, 1] and len(c._free) == 7
    c.free(0)
    assert len(c._free) == 8 and c.table[1, :2].tolist() == c._pages[1]
    c.free(1)
    assert len(c._free) == 9
    with pytest.raises(AssertionError, match="more steps"):
        c.advance_host_step()
    c.free(2)
    assert sorted(c._free) == list(range(10)) and c._holders == [0] * 10


@pytest.mark.parametrize("more,message", [
    (dict(num_layers=0), "needs layers"), (dict(num_q_heads=3, num_kv_heads=2), "multiple"), (dict(num_q_heads=17), "more than 16"), (dict(head_dim=96), "head_dim"),
    (dict(page_size=24), "page_size"), (dict(page_size=8), "page_size"), (dict(sink_len=-1), "negative"), (dict(window=-1), "negative"), (dict(num_pages=0), "needs a page"),
    (dict(sections=(16, 16)), "inv_freq"),
])
def test_caches_that_cannot_be_are_refused(more, message):
    with pytest.raises(AssertionError, match=message):
        cache(**more)


def test_refused_calls_leave_the_cache_as_it_was():
    c = cache()
    for call in (lambda: c.prefill_update_kv_cache(bf(3, 101, 1, 64), bf(3, 101, 1, 64), 0), lambda: c.prefill_update_kv_cache(bf(3, 0, 1, 64), bf(3, 0, 1, 64), 0),
                 lambda: c.prefill_update_kv_cache(bf(2, 5, 1, 64), bf(2, 5, 1, 64), 0), lambda: c.prefill_update_kv_cache(bf(3, 5, 1, 64), bf(3, 5, 1, 64), 0, lens=[1, 2]),
                 lambda: c.prefill_update_kv_cache(bf(3, 5, 1, 64), bf(3, 5, 1, 64), 0, lens=[1, 2, 6]),
                 lambda: c.extend_attention(0, bf(3, 2, 2, 32), bf(3, 2, 1, 64), bf(3, 2, 1, 64)), lambda: c.extend_attention(0, bf(3, 2, 2, 64), bf(3, 1, 1, 64), bf(3, 2, 1, 64)),
                 lambda: c.extend_attention(0, bf(3, 2, 2, 64), bf(3, 2, 1, 64), bf(3, 2, 1, 64), lens=[3, 0, 0]),
                 lambda: c.extend_attention(0, bf(3, 101, 2, 64), bf(3, 101, 1, 64), bf(3, 101, 1, 64)), lambda: c.decode_attention(1, bf(3, 2, 64), bf(3, 1, 1, 64), bf(3, 1, 1, 64))):
        with pytest.raises(AssertionError):
            call()
        assert c._lens == [0, 0, 0] and c.lens.tolist() == [0, 0, 0] and len(c._free) == c.num_pages


# ---- the plain form -------------------------------------------------------------------------------------------------

def test_the_plain_rotation_keeps_lengths_and_goes_by_differences():
    g = torch.Generator().manual_seed(0)
    x, y = (torch.randn((5, 1, 16), generator=g, dtype=torch.float64) for _ in range(2))
    inv = 100.0 ** (-torch.arange(8) / 8)
    p = torch.tensor([[0], [3], [7], [100], [2 ** 30]])
    for inter in (False, True):
        a, b = ref.rotate(x, p, inv, inter), ref.rotate(y, p, inv, inter)
        assert torch.allclose((a * b).sum(-1), (x * y).sum(-1)) and torch.equal(a[0], x[0])
        shift = ref.rotate(x, p + 11, inv, inter), ref.rotate(y, p + 11, inv, inter)
        assert torch.allclose((shift[0] * b).sum(-1)[1:4], (ref.rotate(x, p * 0 + 11, inv, inter) * y).sum(-1)[1:4])
    axes = torch.stack([p[:, 0], p[:, 0]], -1)
    assert torch.equal(ref.rotate(x, axes, inv, sections=(3, 5)), ref.rotate(x, p, inv))


def test_the_plain_rows_and_spans():
    assert ref.attended(5, [0, 1], 4, 2, 8) == [0, 1, 2, 3, 4, 5]
    assert ref.attended(5, [7, 1], 4, 2, 8) == [4, 5] and ref.attended(9, [0, 1], 4, 2, 7) == list(range(7))
    assert ref.attended(6, [0, 1], 4, 2, 8, n_sink=1, window=3) == [0, 4, 5, 6]
    assert ref.spans(2, [-3, 1 << 31], None, [9, -1], 4, 8) == [(0, 4, 0), (4, 0, 1 << 30)]
    assert ref.spans(3, None, [-2, 3, 1, 99], None, 2, 8) == [(0, 2, 0), (3, 0, 0), (1, 2, 0)]


@pytest.mark.parametrize("source,kernels", [("paged.hip", ["paged_append_kernel"]), ("paged_attn.hip", ["paged_rows_kernel", "paged_join_kernel"]),
                                            ("paged_chunk.hip", ["paged_chunk_kernel", "paged_chunk_join_kernel"])])
def test_kernels_do_not_spill(source, kernels):
    """The 256-column kernels stand at the 256 registers that two waves to a SIMD leave: 16 spilled ones made a chunk's take 1.4 times as long."""
    from test_host_logic import test_scan_kernels_do_not_spill as check
    check(source, kernels)
