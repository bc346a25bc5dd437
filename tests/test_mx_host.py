"""The block-scaled cache without a GPU: the plain form's own properties, struct layouts, and every refusal."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

from diffcache_amd import _hip as hip
from oracle import mx as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("bits", [4, 8])
def test_the_plain_form_holds_what_the_format_can(bits):
    """Numbers of the grid times a power of two come back as they went in; others within half a step of the format."""
    rng = np.random.default_rng(bits)
    g = ref.grid(bits)
    g = g[np.isfinite(g)]
    x = rng.choice(g, (200, 64))
    x[:, 0] = x[:, 32] = g.max()
    x = x * np.ldexp(1.0, rng.integers(-100, 100, (200, 1)))
    assert np.array_equal(ref.decode(*ref.encode(x, bits)), x)
    y = rng.standard_normal((300, 128))
    held = ref.decode(*ref.encode(y, bits))
    most = np.abs(y).reshape(300, 4, 32).max(-1).repeat(32, -1)
    assert (np.abs(held - y) <= most / (3.5 if bits == 4 else 14.5)).all()
    assert np.abs(held - y).mean() < (0.12 if bits == 4 else 0.03)


def test_scales_of_small_large_and_unbounded_blocks():
    x = np.zeros((6, 64))
    x[1, :32], x[2, 3], x[3, 40], x[4, 0], x[5, :] = 3.3e38, np.inf, np.nan, 1e-38, 2.0 ** -133
    for bits, (lo, hi) in ref.LIMITS.items():
        codes, scale = ref.encode(x, bits)
        held = ref.decode(codes, scale)
        assert scale[0].tolist() == [lo, lo] and scale[1, 0] == hi and scale[2].tolist() == [255, lo] and scale[3, 1] == 255
        assert held[1, 0] == (6 * 2.0 ** 125 if bits == 4 else 448 * 2.0 ** 119)
        assert np.isnan(held[2, :32]).all() and np.isnan(held[3, 32:]).all() and not np.isnan(held[3, :32]).any()
        assert scale[5, 0] == lo


@pytest.mark.parametrize("name,cls", [("dc_mx_store", hip.MxStoreArgs), ("dc_mx_attn_args", hip.MxAttnArgs)])
def test_structs_match_the_header(name, cls):
    header = open(os.path.join(ROOT, "include", "diffcache_hip.h")).read()
    body = header[header.index("typedef struct %s {" % name):header.index("} %s;" % name)]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
    names = [re.sub(r"[^A-Za-z0-9_]", "", n.split()[-1]) for decl in body.split(";") if decl.strip()
             for n in decl.replace("*", " ").split(",")]
    assert names == [n for n, _ in cls._fields_]
    packed = hip._MX_STORE if cls is hip.MxStoreArgs else hip._MX_ATTN
    assert packed.size == ctypes.sizeof(cls)


def test_packed_bytes_are_the_structs():
    store = hip._MX_STORE.pack(*range(1, 7), 4, 99)
    assert store == bytes(hip.MxStoreArgs(*range(1, 7), 4, 99))
    other = hip._MX_STORE.pack(*range(11, 17), 8, 98)
    args = hip._MX_ATTN.pack(*range(21, 27), store, other, 31, 32, *range(41, 48), 0.25)
    want = hip.MxAttnArgs(*range(21, 27), hip.MxStoreArgs.from_buffer_copy(store), hip.MxStoreArgs.from_buffer_copy(other), 31,
                          32, *range(41, 48), 0.25)
    assert args == bytes(want)


def fake(bits=4, n_rows=64, hd=128, **more):
    """A store that no kernel is launched on: every call below is refused first."""
    s = hip.MxStoreArgs(1 << 20, 1 << 21, 2 * n_rows * hd * bits // 8, n_rows * hd * bits // 8, 2 * n_rows * (hd // 32),
                        n_rows * (hd // 32), bits, n_rows)
    for name, x in more.items():
        setattr(s, name, x)
    return s


def ref_of(x):
    """A struct as the library's calls take it."""
    return bytes(x)


def refused(rc, message):
    assert rc == -22 and re.search(message, hip.lib.dc_last_error().decode()), (rc, hip.lib.dc_last_error())


BAD_STORES = [
    (dict(bits=5), "5 bits"), (dict(bits=0), "0 bits"), (dict(codes=None), "null"), (dict(scale=None), "null"),
    (dict(codes=(1 << 20) + 8), "16-byte"), (dict(code_batch_stride=72), "16 bytes"), (dict(code_head_stride=8), "16 bytes"),
    (dict(scale=(1 << 21) + 2), "multiples of 4"), (dict(scale_head_stride=6), "multiples of 4"), (dict(code_batch_stride=-64), "negative"),
    (dict(scale_head_stride=-4), "negative"), (dict(n_rows=-1), "negative"),
]


@pytest.mark.parametrize("change,message", BAD_STORES)
def test_bad_stores_are_refused_everywhere(change, message):
    good, bad = fake(), fake(**change)
    p = 1 << 22
    for k, v in ((good, bad), (bad, good)):
        refused(hip.lib.dc_mx_ingest_bf16(ref_of(k), ref_of(v), p, p, None, 2, 8, 2, 128, 0, *[1024] * 6, None), message)
        refused(hip.lib.dc_mx_append_bf16(ref_of(k), ref_of(v), p, p, p, 2, 2, 128, None), message)
        refused(hip.lib.dc_mx_gather_rows_bf16(ref_of(k), ref_of(v), None, p, p, 2, 2, 8, 0, 128, 0, 1024, 1024, 128, None), message)
        a = attn_args(k=k, v=v)
        refused(hip.lib.dc_mx_attn_bf16(ref_of(a), None), message)


def attn_args(**change):
    p = 1 << 22
    a = hip.MxAttnArgs(p, None, None, p, None, p, fake(), fake(), p, 1 << 30, 2, 2, 4, 128, 64, 0, 0, 0.1)
    for name, x in change.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("change,message", [
    (dict(q=None), "null"), (dict(out=None), "null"), (dict(new_k=1 << 22), "both"), (dict(new_v=1 << 22), "both"), (dict(group=0), "group"),
    (dict(group=17), "group"), (dict(hd=96), "head_dim"), (dict(n_rows=65), "outside"), (dict(n_rows=-1), "outside"),
    (dict(n_sink=-1), "negative"), (dict(window=-1), "negative"), (dict(q=(1 << 22) + 2), "aligned"), (dict(n_h=0), "bad sizes"),
    (dict(n_b=-1), "bad sizes"), (dict(n_b=1 << 23), "too many units"), (dict(k=fake(n_rows=4096), v=fake(n_rows=4096), n_rows=4096, workspace=None), "workspace"),
    (dict(k=fake(n_rows=4096), v=fake(n_rows=4096), n_rows=4096, workspace=(1 << 22) + 16), "workspace"),
    (dict(new_k=1 << 22, new_v=(1 << 22) + 8), "aligned"),
    (dict(new_k=1 << 22, new_v=1 << 22, k=fake(code_batch_stride=0)), "share"),
    (dict(new_k=1 << 22, new_v=1 << 22, v=fake(scale_head_stride=0)), "share"),
])
def test_bad_attention_is_refused(change, message):
    a = attn_args(**change)
    refused(hip.lib.dc_mx_attn_bf16(ref_of(a), None), message)


def test_a_small_workspace_is_refused():
    a = attn_args(k=fake(n_rows=4096), v=fake(n_rows=4096), n_rows=4096, workspace_bytes=1024)
    assert hip.lib.dc_mx_attn_bf16(ref_of(a), None) == -12
    assert "needed" in hip.lib.dc_last_error().decode()
    refused(hip.lib.dc_mx_attn_bf16(None, None), "null")


def test_enough_workspace_for_more_is_enough_for_fewer():
    for hd in (64, 128, 256):
        last = 0
        for units in (1, 2, 7, 64, 300, 512, 513, 5000):
            sizes = [hip.mx_attn_workspace_bytes(units, 4, hd, n) for n in (0, 1, 64, 65, 1000, 100000, 2**31 - 1)]
            assert sizes == sorted(sizes) and sizes[-1] >= last
            last = sizes[-1]
    assert hip.mx_attn_workspace_bytes(0, 4, 128, 100) == hip.mx_attn_workspace_bytes(4, 4, 128, -1) == 0


def test_bad_rows_are_refused():
    s, p = fake(), 1 << 22
    call = lambda **c: hip.lib.dc_mx_ingest_bf16(*{**dict(k=ref_of(s), v=ref_of(s), ks=p, vs=p, lens=None, b=2, seq=8, h=2, hd=128, at=0, s0=1024, s1=1024,  # noqa: E731
                                                          s2=1024, s3=1024, s4=1024, s5=1024, st=None), **c}.values())
    refused(call(k=None), "null")
    refused(call(ks=None), "null")
    refused(call(vs=p + 8), "aligned")
    refused(call(at=60), "outside")
    refused(call(at=-1), "bad sizes")
    refused(call(seq=-1), "bad sizes")
    refused(call(s1=1028), "multiples of 8")
    refused(call(s5=4), "multiples of 8")
    refused(call(hd=32), "head_dim")
    assert call(seq=0) == 0 and call(b=0) == 0
    call = lambda **c: hip.lib.dc_mx_gather_rows_bf16(*{**dict(k=ref_of(s), v=ref_of(s), idx=None, ok=p, ov=p, b=2, h=2, n=8, ist=8, hd=128, off=0,  # noqa: E731
                                                               d0=1024, d1=1024, d2=128, st=None), **c}.values())
    refused(call(ok=None, ov=None), "null")
    refused(call(k=None), "source missing")
    refused(call(idx=p, ist=7), "idx_unit_stride")
    refused(call(ov=p + 2), "aligned")
    refused(call(d2=130), "multiples of 8")
    refused(call(off=-1), "bad sizes")
    refused(call(n=-1), "bad sizes")
    assert call(n=0) == 0 and call(b=0) == 0
    refused(hip.lib.dc_mx_append_bf16(ref_of(s), ref_of(s), p, p, None, 2, 2, 128, None), "null")
    refused(hip.lib.dc_mx_append_bf16(ref_of(s), ref_of(s), p + 8, p, p, 2, 2, 128, None), "aligned")


def test_wrappers_refuse_what_does_not_fit():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    with pytest.raises(hip.DiffCacheError, match="GPU memory"):
        hip.MxStore(u8(1, 2, 8, 64), u8(1, 2, 8, 4))
    with pytest.raises(hip.DiffCacheError, match="GPU memory"):
        hip.MxStore.zeros(1, 2, 8, 128, 4, "cpu")
    for codes, scale in ((u8(1, 2, 8, 64), u8(1, 2, 7, 4)), (u8(2, 8, 64), u8(2, 8, 4)), (u8(1, 2, 8, 64).float(), u8(1, 2, 8, 4))):
        with pytest.raises(hip.DiffCacheError, match="uint8 tensors"):
            hip.MxStore(codes, scale)
    with pytest.raises(hip.DiffCacheError, match="neither 4 nor 8 bits"):
        hip.MxStore(u8(1, 2, 8, 96), u8(1, 2, 8, 4))
    for codes, scale in ((u8(1, 2, 64, 8).transpose(2, 3), u8(1, 2, 8, 4)), (u8(1, 8, 2, 64).transpose(1, 2), u8(1, 2, 8, 4)),
                         (u8(1, 2, 8, 64), u8(1, 8, 2, 4).transpose(1, 2)), (u8(1, 2, 8, 64), u8(1, 2, 8, 8)[..., :4])):
        with pytest.raises(hip.DiffCacheError, match="one after another"):
            hip.MxStore(codes, scale)
    for bits, hd in ((5, 128), (4, 96)):
        with pytest.raises(hip.DiffCacheError, match="not supported"):
            hip.MxStore.zeros(1, 1, 1, hd, bits, "cpu")
