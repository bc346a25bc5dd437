"""Attention over the block-scaled cache in one part of four waves, in few parts and in many: every way in which units and steps are
dealt to blocks, with the number of parts looked at, and the join in captured steps."""
import math
import re

import numpy as np
import pytest
import torch

from oracle import mx as ref
from test_gpu_mx import bf16, check_attention, f64, held, hip, keys, store_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def needed(q, ks, vs, n_rows, n_sink=0, window=0):
    """Workspace bytes of a call, by the refusal of a small one; 0 where it takes none."""
    try:
        hip().mx_attn(q, ks, vs, n_rows=n_rows, n_sink=n_sink, window=window, workspace=torch.empty(256, dtype=torch.uint8, device=DEV))
    except hip().DiffCacheError as e:
        return int(re.search(r"< (\d+) needed", str(e)).group(1))
    return 0


def parts(q, ks, vs, n_rows=None, n_sink=0, window=0):
    """Parts that a unit is cut into."""
    b, h, n, hd = ks.shape
    n = min(n, vs.shape[2]) if n_rows is None else n_rows
    bytes_, group = needed(q, ks, vs, n, n_sink, window), q.numel() // (b * h * hd)
    up = lambda x: (x + 255) // 256 * 256  # noqa: E731
    found = [p for p in range(2, 1025) if up(b * h * p * group * hd * 4) + up(b * h * p * group * 8) == bytes_]
    assert bytes_ == 0 or len(found) >= 1, bytes_
    assert bytes_ <= hip().mx_attn_workspace_bytes(b * h, group, hd, n)
    return found[0] if bytes_ else 1


def filled(rng, b, h, n, hd, bits, like_keys, room=None):
    """A store written by mx_ingest (long ones take numpy too long); rows behind n hold what must not be read."""
    room = n if room is None else room
    s = hip().MxStore(torch.full((b, h, room, hd * bits // 8), 0xff, dtype=torch.uint8, device=DEV),
                      torch.full((b, h, room, hd // 32), 0xff, dtype=torch.uint8, device=DEV))
    g = torch.Generator(device=DEV).manual_seed(int(rng.integers(1 << 30)))
    x = torch.randn((b, n, h, hd), generator=g, device=DEV)
    if like_keys:
        x *= torch.exp(torch.randn(hd, generator=g, device=DEV))
    x = x.to(torch.bfloat16)
    hip().mx_ingest(s, s, x, x)
    return s


def shared(s, b):
    return hip().MxStore(s.codes.expand(b, -1, -1, -1), s.scale.expand(b, -1, -1, -1))


# ---- how units and rows are dealt out -----------------------------------------------------------------------------------

@pytest.mark.parametrize("b,h,g,hd,bits,n,want", [
    (260, 2, 2, 64, (4, 4), 1700, 1),        # more units than places
    (150, 2, 1, 128, (8, 4), 1800, 1),       # between a half of them and all
    (129, 2, 3, 256, (4, 8), 900, 1),
    (100, 2, 4, 128, (4, 4), 1700, 2), (60, 2, 4, 64, (4, 8), 2500, 4), (43, 4, 2, 128, (4, 4), 1601, 2),
])
def test_many_units(b, h, g, hd, bits, n, want):
    """A prefix that all sequences share, of another length in each."""
    rng = np.random.default_rng(n + b)
    one = store_of(keys(rng, (1, h, n, hd)), bits[0]), store_of(rng.standard_normal((1, h, n, hd)), bits[1])
    ks, vs = (shared(s, b) for s in one)
    q, qx = bf16(rng.standard_normal((b, h * g, hd)))
    assert parts(q, ks, vs) == want
    lens = rng.integers(0, n + 1, b)
    lens[:5] = [n, 0, 1, n - 1, 64]
    check_attention(q, qx, ks, vs, lens.tolist())


def test_many_units_and_a_token():
    """One part of four waves to a unit, and the token's row written by the wave with the last step."""
    rng = np.random.default_rng(1)
    b, h, g, hd, n = 260, 2, 2, 64, 1700
    ks, vs = filled(rng, b, h, n - 1, hd, 4, True, n), filled(rng, b, h, n - 1, hd, 8, False, n)
    q, qx = bf16(rng.standard_normal((b, h * g, hd)))
    nk, nv = (bf16(rng.standard_normal((b, h, hd)))[0] for _ in range(2))
    assert parts(q, ks, vs) == 1
    lens = rng.integers(0, n, b)
    lens[:4] = [n - 1, n, 0, 63]
    at = torch.from_numpy(lens.astype(np.int32)).to(DEV)
    kept = [hip().MxStore(s.codes.clone(), s.scale.clone()) for s in (ks, vs)]
    hip().mx_append(*kept, nk, nv, at)
    out = hip().mx_attn(q, ks, vs, at, new_k=nk, new_v=nv)
    for s, w in zip((ks, vs), kept):
        assert torch.equal(s.codes, w.codes) and torch.equal(s.scale, w.scale)
    lens = np.minimum(lens + 1, n)
    lens[1] = n - 1                            # (its last row is not written)
    few = slice(0, 40)
    want = check_attention(q[few], qx[few], *(hip().MxStore(s.codes[few], s.scale[few]) for s in kept), lens[few].tolist())[0]
    rows = [0, 2, 3]
    assert (out[rows].double() - want[rows].double()).abs().max() <= 2.0 ** -7 * want[rows].double().abs().max()
    same = hip().mx_attn(q, *kept, torch.from_numpy(lens.astype(np.int32)).to(DEV))
    rows = [i for i in range(b) if i != 1]
    assert torch.equal(out[rows], same[rows])


@pytest.mark.parametrize("b,h,g,n,want", [(64, 2, 2, 6200, 8), (24, 8, 4, 4100, 5), (512, 2, 1, 1700, 1)])
def test_lean_rows_of_many_units(b, h, g, n, want):
    """64 columns in 4 bits from 12288 steps on: up to 1024 blocks."""
    rng = np.random.default_rng(n)
    assert b * h * ((n + 63) // 64) >= 6 * 4 * 512
    one = store_of(keys(rng, (1, h, n, 64)), 4), store_of(rng.standard_normal((1, h, n, 64)), 4)
    ks, vs = (shared(s, b) for s in one)
    q, qx = bf16(rng.standard_normal((b, h * g, 64)))
    assert parts(q, ks, vs) == want
    lens = rng.integers(0, n + 1, b)
    lens[:4] = [n, 0, 1, n - 1]
    check_attention(q, qx, ks, vs, lens.tolist())


@pytest.mark.parametrize("hd,bits,g,n,want", [(64, (4, 4), 2, 12288 * 64, 1024), (64, (4, 4), 1, 12288 * 64 - 100, 512), (128, (4, 4), 4, 300001, 512),
                                              (256, (8, 4), 2, 100003, 512)])
def test_one_unit_in_many_parts(hd, bits, g, n, want):
    rng = np.random.default_rng(hd)
    ks, vs = filled(rng, 1, 1, n, hd, bits[0], True, n + 7), filled(rng, 1, 1, n, hd, bits[1], False, n + 7)
    q, qx = bf16(rng.standard_normal((1, g, hd)))
    assert parts(q, ks, vs, n) == want
    for length in (n, n - 1, 1, 70001):
        check_attention(q, qx, ks, vs, [length], n_rows=n)


# ---- sinks and a window in parts ----------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,bits,g", [(64, (4, 4), 7), (128, (4, 4), 4), (128, (8, 8), 16), (256, (8, 4), 3)])
@pytest.mark.parametrize("n_sink,window", [(4, 2100), (700, 2100), (1, 2047), (65, 3001), (2500, 2300), (0, 1700)])
def test_sinks_and_window_in_parts(hd, bits, g, n_sink, window):
    """In a workspace of exactly the bytes that the call needs, whose surroundings stay as they are; with a token too."""
    rng = np.random.default_rng(n_sink + window)
    n, h = 5000, 2
    lens = [5000, 4999, 0, 1, window + n_sink, window + n_sink + 1, window + n_sink - 1, 3300]
    lens = [min(x, n) for x in lens]
    b = len(lens)
    x, y = keys(rng, (1, h, n, hd)), rng.standard_normal((1, h, n, hd))
    one = store_of(x, bits[0]), store_of(y, bits[1])
    stores = []
    for s in one:
        codes, scale = (t.expand(b, -1, -1, -1).contiguous() for t in (s.codes, s.scale))
        for i, length in enumerate(lens):      # rows between and behind hold what must not be read
            rows = np.setdiff1d(np.arange(n), ref.attended(length, n_sink, window))
            codes[i, :, rows], scale[i, :, rows] = 0xff, 0xff
        stores.append(hip().MxStore(codes, scale))
    ks, vs = stores
    q, qx = bf16(rng.standard_normal((b, h * g, hd)))
    bytes_ = needed(q, ks, vs, n, n_sink, window)
    assert parts(q, ks, vs, n, n_sink, window) > 1
    room = torch.full((bytes_ + 8192,), 0xa5, dtype=torch.uint8, device=DEV)
    ws = room[4096:4096 + bytes_]
    assert ws.data_ptr() % 256 == 0
    first, _ = check_attention(q, qx, ks, vs, lens, n_sink=n_sink, window=window, workspace=ws)
    assert (room[:4096] == 0xa5).all() and (room[4096 + bytes_:] == 0xa5).all()
    # the last attended row written on the way gives the same, bit for bit
    at = torch.tensor([max(x - 1, 0) for x in lens], dtype=torch.int32, device=DEV)
    nk, nv = hip().mx_gather_rows(ks, vs, at.view(b, 1).expand(b, h).reshape(b * h, 1).contiguous())
    live = [i for i in range(b) if lens[i]]
    for s in (ks, vs):
        for i in live:
            s.codes[i, :, lens[i] - 1], s.scale[i, :, lens[i] - 1] = 0xff, 0xff
    nk, nv = (t.view(b, h, hd).contiguous() for t in (nk, nv))
    out = hip().mx_attn(q, ks, vs, at, new_k=nk, new_v=nv, n_sink=n_sink, window=window, workspace=ws)
    assert torch.equal(out[live], first[live])
    assert (room[:4096] == 0xa5).all() and (room[4096 + bytes_:] == 0xa5).all()


# ---- parts in captured steps --------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,bits,n_sink,window", [(128, (4, 4), 0, 0), (64, (4, 4), 0, 0), (256, (8, 4), 5, 2100)])
def test_captured_steps_in_parts(hd, bits, n_sink, window):
    """Two graphs with a workspace each, replayed at once on two streams and among eager work: every replay against an eager step."""
    rng = np.random.default_rng(hd)
    b, h, g, n = 2, 2, 4, 4000
    k, v = keys(rng, (b, h, n, hd)), rng.standard_normal((b, h, n, hd))
    runs = []
    for start in ([3990, 1600], [0, 2900]):
        c = dict(ks=store_of(k, bits[0]), vs=store_of(v, bits[1]), lens=torch.tensor(start, dtype=torch.int32, device=DEV), start=start)
        c["eager"] = (store_of(k, bits[0]), store_of(v, bits[1]))
        for name, shape in (("q", (b, h * g, hd)), ("nk", (b, h, hd)), ("nv", (b, h, hd)), ("out", (b, h * g, hd))):
            c[name] = torch.zeros(shape, dtype=torch.bfloat16, device=DEV)
        c["lse"] = torch.empty((b, h * g), device=DEV)
        assert parts(c["q"], c["ks"], c["vs"], n, n_sink, window) > 1
        c["ws"] = torch.empty(needed(c["q"], c["ks"], c["vs"], n, n_sink, window), dtype=torch.uint8, device=DEV)
        c["stream"], c["graph"] = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        c["stream"].wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(c["graph"], stream=c["stream"]):
            hip().mx_attn(c["q"], c["ks"], c["vs"], c["lens"], new_k=c["nk"], new_v=c["nv"], out=c["out"], lse=c["lse"], workspace=c["ws"],
                          n_sink=n_sink, window=window)
            c["lens"].add_(1)
        runs.append(c)
    for i in range(8):
        for c in runs:
            for name in ("q", "nk", "nv"):
                c[name].copy_(torch.randn(c[name].shape, device=DEV))
        for c in runs:
            c["stream"].wait_stream(torch.cuda.current_stream())
        for c in runs:
            with torch.cuda.stream(c["stream"]):
                c["graph"].replay()
        for c in runs:
            torch.cuda.current_stream().wait_stream(c["stream"])
        if i % 2:
            torch.cuda.synchronize()
        for c in runs:
            lens = torch.tensor([x + i for x in c["start"]], dtype=torch.int32, device=DEV)
            out, lse = hip().mx_attn(c["q"], *c["eager"], lens, new_k=c["nk"], new_v=c["nv"], n_sink=n_sink, window=window, want_lse=True)
            assert torch.equal(c["out"], out) and torch.equal(c["lse"], lse), i
            assert torch.equal(c["lens"], lens + 1)
            for s, w in zip((c["ks"], c["vs"]), c["eager"]):
                assert torch.equal(s.codes, w.codes) and torch.equal(s.scale, w.scale)


def test_a_captured_step_of_a_cache_in_parts():
    """MxCache beyond the lengths that one kernel takes: captured for max_length and replayed from a short prompt past several cuts."""
    from diffcache_amd import MxCache
    layers, b, h, g, hd, room = 2, 2, 2, 4, 128, 2600
    caches = [MxCache(layers, b, room, h, h * g, hd, key_bits=8) for _ in range(2)]
    gen = torch.Generator(device=DEV).manual_seed(1)
    for layer in range(layers):
        k, v = (torch.randn((b, 2560, h, hd), generator=gen, device=DEV).to(torch.bfloat16) for _ in range(2))
        for c in caches:
            c.prefill_update_kv_cache(k, v, layer, lens=[2560, 1490])
    captured, eager = caches
    q, nk, nv = (torch.zeros((b, x, hd), dtype=torch.bfloat16, device=DEV) for x in (h * g, h, h))
    assert parts(q, captured.kstore[0], captured.vstore[0]) > 1
    outs = [torch.empty_like(q) for _ in range(layers)]
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        for layer in range(layers):
            captured.decode_attention(layer, q, nk, nv, out=outs[layer])
    for step in range(40):
        for t in (q, nk, nv):
            t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        graph.replay()
        captured.advance_host_step()
        for layer in range(layers):
            out = eager.decode_attention(layer, q, nk, nv)
            # (the two may cut the rows otherwise: sums in another order.  Each is within 2^-8 of its own, and of 2^-13 of the weighted
            # |v| of at most 6 for P, exp2 and fp32 sums)
            assert ((out.double() - outs[layer].double()).abs() <= 2.0 ** -7 * out.double().abs() + 2.0 ** -12 * 6).all(), (step, layer)
    assert torch.equal(captured.lens, eager.lens) and captured.seq_len(0) == 2600
    for x, y in zip(captured.kstore + captured.vstore, eager.kstore + eager.vstore):
        assert torch.equal(x.codes, y.codes) and torch.equal(x.scale, y.scale)


# ---- large logits -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd,bits,group,n", [(64, 4, 4, 300), (128, 4, 7, 5000), (128, 8, 16, 2000), (256, 8, 2, 3000)])
@pytest.mark.parametrize("scale", [1.0, 4.0, -2.0])
def test_large_logits(hd, bits, group, n, scale):
    """Whole numbers whose products and sums fp32 holds exactly, to about 10^4: what is left is the rounding of a logit's two factors of
    scale log2(e), 2^-24 of it each, and of its difference from the maximum."""
    rng = np.random.default_rng(n)
    grid = np.array([-6.0, -4, -3, -2, -1, 0, 1, 2, 3, 4, 6])
    kx, vx = rng.choice(grid, (1, 1, n, hd)), rng.choice(grid, (1, 1, n, hd))
    kx[..., ::32] = vx[..., ::32] = 6          # (so that every block's scale is 1)
    qx = rng.integers(-16, 17, (1, group, hd)).astype(float)
    q = torch.from_numpy(qx).to(torch.bfloat16).to(DEV)
    ks, vs = store_of(kx, bits), store_of(vx, bits)
    assert np.array_equal(held(ks), kx) and np.array_equal(held(vs), vx)
    out, lse = hip().mx_attn(q, ks, vs, scale=scale, want_lse=True)
    want, want_lse, weight, _ = ref.attention(qx[0], kx[0, 0], vx[0, 0], scale)
    logit = np.abs(qx[0] @ kx[0, 0].T * scale).max(1)
    assert logit.max() > 600
    d = 3 * 2.0 ** -24 * logit
    rel = 2 * d + 2.0 ** -16 + 2.0 ** -21 + 2 * n * 2.0 ** -24
    # Far from the maximum e^x is below 2^-126, the least normal number of fp32 and of bf16: a weight and what P's second number has of it
    # may be 0, each off by 2^-126 times |v| <= 6, over a sum of 1 or more; so may the output: n (12 2^-126) + 2^-126 < n 2^-122.
    tol = 2.0 ** -8 * np.abs(want) + weight * (rel * (1 + 2.0 ** -7))[:, None] + n * 2.0 ** -122
    assert (np.abs(want) > 4 * tol).mean() > 0.8   # (no other output passes)
    assert (np.abs(f64(out)[0] - want) <= tol).all()
    assert (np.abs(f64(lse)[0] - want_lse) <= d + 2.0 ** -20 + n * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(want_lse)).all()
    assert math.isclose(float(lse.abs().max()), np.abs(want_lse).max(), rel_tol=1e-5)
