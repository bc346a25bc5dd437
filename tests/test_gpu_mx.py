"""The cache in blocks of 32 numbers on the GPU: codes and scales byte for byte, rows read back exactly, attention against 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import mx as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def hip():
    from diffcache_amd import _hip
    return _hip


def bf16(x):
    """numpy float64 -> torch bf16 on the GPU and the same numbers in float64."""
    t = torch.from_numpy(np.asarray(x, dtype=np.float32)).to(torch.bfloat16)
    return t.to(DEV), t.double().numpy()


def f64(t):
    return t.detach().cpu().double().numpy()


def keys(rng, shape):
    return rng.standard_normal(shape) * np.exp(rng.standard_normal(shape[-1:]))


def store_of(x, bits, room=None):
    """A store that holds x (b, h, n, hd), rows behind n filled with what must not be read (NaN scales, all bits set)."""
    b, h, n, hd = x.shape
    room = n if room is None else room
    codes = np.full((b, h, room, hd * bits // 8), 0xff, np.uint8)
    scale = np.full((b, h, room, hd // 32), 0xff, np.uint8)
    codes[:, :, :n], scale[:, :, :n] = ref.encode(x, bits)
    return hip().MxStore(torch.from_numpy(codes).to(DEV), torch.from_numpy(scale).to(DEV))


def held(store):
    return ref.decode(store.codes.cpu().numpy(), store.scale.cpu().numpy())


# ---- the format -----------------------------------------------------------------------------------------------------

def all_bf16(seed):
    """Every bf16 bit pattern in some block: in order (neighbours of one size together) and shuffled, (1, n, 1, 64)."""
    w = np.arange(65536, dtype=np.uint16)
    if seed:
        np.random.default_rng(seed).shuffle(w)
    return torch.from_numpy(w.view(np.int16).copy()).view(torch.bfloat16).view(1, 1024, 1, 64)


def ties(bits):
    """Blocks around every boundary between two codes, and around the one at which the scale moves, for several exponents."""
    g = ref.grid(bits)[:ref.LAST[bits] + 1]
    edges = np.concatenate([(g[1:] + g[:-1]) / 2, [g[-1] + (g[-1] - g[-2]) / 2]])
    rows = []
    for e in (-100, -3, 0, 1, 40, 110):
        for top in (g[-1], g[-1] * 0.51, edges[-1], np.nextafter(np.float32(edges[-1]), 0)):
            for part in np.array_split(np.concatenate([edges, -edges]), max(1, 2 * len(edges) // 31)):
                x = np.zeros(64)
                x[:len(part)] = np.where(np.abs(part) <= top, part, 0)
                x[31] = x[63] = top
                rows.append(np.ldexp(x, e))
    return torch.from_numpy(np.array(rows, dtype=np.float32)).to(torch.bfloat16).view(1, -1, 1, 64)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("src", ["in order", "shuffled", "ties"])
def test_codes_and_scales_byte_for_byte(bits, src):
    x = ties(bits) if src == "ties" else all_bf16(0 if src == "in order" else 5)
    n = x.shape[1]
    s = hip().MxStore.zeros(1, 1, n, 64, bits, DEV)
    hip().mx_ingest(s, s, x.to(DEV), x.to(DEV))
    codes, scale = ref.encode(x.double().numpy()[0, :, 0], bits)
    assert np.array_equal(s.scale.cpu().numpy()[0, 0], scale)
    got = s.codes.cpu().numpy()[0, 0]
    nan = np.repeat(scale == 255, 32 * bits // 8, axis=-1)
    assert np.array_equal(np.where(nan, 0, got), np.where(nan, 0, codes)) and not got[nan].any()
    # what is held, in bf16: exact, and within the format's step of what came
    back, _ = hip().mx_gather_rows(s, None)
    want = ref.decode(codes, scale)
    assert np.array_equal(f64(back)[0, 0], want, equal_nan=True)
    assert np.isfinite(want[~np.repeat(scale == 255, 32, axis=-1)]).all()
    inside = (np.repeat(scale, 32, axis=-1) > ref.LIMITS[bits][0]) & (np.repeat(scale, 32, axis=-1) < ref.LIMITS[bits][1])
    step = np.ldexp(1.0 if bits == 4 else 16.0, np.repeat(scale, 32, axis=-1).astype(int) - 127)
    assert (np.abs(want - x.double().numpy()[0, :, 0])[inside] <= step[inside]).all()


# ---- writing and reading back -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kbits,vbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("b,h,seq,dst", [(1, 1, 1, 0), (2, 3, 5, 2), (1, 2, 63, 0), (3, 1, 257, 7), (2, 2, 1030, 1)])
def test_prompt_rows(hd, kbits, vbits, b, h, seq, dst):
    rng = np.random.default_rng(hash((hd, kbits, vbits, seq)) % 2**32)
    (k, kx), (v, vx) = bf16(keys(rng, (b, seq, h, hd))), bf16(rng.standard_normal((b, seq, h, hd)))
    room = dst + seq + 3
    ks, vs = (hip().MxStore(torch.full((b, h, room, hd * bits // 8), 0x5a, dtype=torch.uint8, device=DEV),
                            torch.full((b, h, room, hd // 32), 100, dtype=torch.uint8, device=DEV)) for bits in (kbits, vbits))
    hip().mx_ingest(ks, vs, k, v, dst_pos=dst)
    for s, x, bits in ((ks, kx, kbits), (vs, vx, vbits)):
        codes, scale = ref.encode(x.transpose(0, 2, 1, 3), bits)
        got_c, got_s = s.codes.cpu().numpy(), s.scale.cpu().numpy()
        assert np.array_equal(got_c[:, :, dst:dst + seq], codes) and np.array_equal(got_s[:, :, dst:dst + seq], scale)
        for rows in (slice(0, dst), slice(dst + seq, None)):          # the others were left as they were
            assert (got_c[:, :, rows] == 0x5a).all() and (got_s[:, :, rows] == 100).all()
    back = hip().mx_gather_rows(ks, vs, row_offset=dst, n_idx=seq)
    for t, s in zip(back, (ks, vs)):
        assert np.array_equal(f64(t), held(s)[:, :, dst:dst + seq])


@pytest.mark.parametrize("lens", [[0, 40, 13], [40, 1, 99], [-3, 39, 0]])
def test_prompts_of_unequal_lengths(lens):
    rng = np.random.default_rng(3)
    b, h, seq, hd = 3, 2, 40, 128
    (k, kx), (v, vx) = bf16(rng.standard_normal((b, seq, h, hd))), bf16(rng.standard_normal((b, seq, h, hd)))
    k[1, 13:] = math.nan                                              # padding may hold anything
    ks, vs = (hip().MxStore(torch.full((b, h, seq, hd * n // 8), 7, dtype=torch.uint8, device=DEV),
                            torch.full((b, h, seq, hd // 32), 9, dtype=torch.uint8, device=DEV)) for n in (4, 8))
    hip().mx_ingest(ks, vs, k, v, lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    kx = f64(k)
    for s, x, bits in ((ks, kx, 4), (vs, vx, 8)):
        codes, scale = ref.encode(x.transpose(0, 2, 1, 3), bits)
        for i, n in enumerate(lens):
            n = min(max(n, 0), seq)
            assert np.array_equal(s.codes.cpu().numpy()[i, :, :n], codes[i, :, :n])
            assert np.array_equal(s.scale.cpu().numpy()[i, :, :n], scale[i, :, :n])
            assert (s.codes.cpu().numpy()[i, :, n:] == 7).all() and (s.scale.cpu().numpy()[i, :, n:] == 9).all()


def test_sources_and_stores_of_other_layouts():
    """Sources (b, h, s, d) transposed and cut out of a fused projection; stores that are views of
    (b, layers, h, rows, .) tensors."""
    rng = np.random.default_rng(4)
    b, h, seq, hd = 2, 3, 37, 128
    k_t, kx = bf16(rng.standard_normal((b, h, seq, hd)))
    qkv, x = bf16(rng.standard_normal((b, seq, 4 * h * hd)))
    v = qkv[..., 2 * h * hd:3 * h * hd].view(b, seq, h, hd)
    vx = x[..., 2 * h * hd:3 * h * hd].reshape(b, seq, h, hd)
    ks, vs = (hip().MxStore(torch.zeros((b, 4, h, 60, hd * n // 8), dtype=torch.uint8, device=DEV)[:, 2, :, 7:57],
                            torch.zeros((b, 4, h, 60, hd // 32), dtype=torch.uint8, device=DEV)[:, 2, :, 7:57]) for n in (4, 8))
    hip().mx_ingest(ks, vs, k_t.transpose(1, 2), v, dst_pos=5)
    for s, want, bits in ((ks, kx, 4), (vs, vx.transpose(0, 2, 1, 3), 8)):
        codes, scale = ref.encode(want, bits)
        assert np.array_equal(s.codes.cpu().numpy()[:, :, 5:42], codes) and np.array_equal(s.scale.cpu().numpy()[:, :, 5:42], scale)
    idx = torch.from_numpy(rng.integers(0, 37, (b * h, 11)).astype(np.int32)).to(DEV)
    big = torch.zeros((b, 20, h, 2, hd), dtype=torch.bfloat16, device=DEV)
    out_k, out_v = big[:, 4:15, :, 0].transpose(1, 2), big[:, 4:15, :, 1].transpose(1, 2)
    got = hip().mx_gather_rows(ks, vs, idx, out_k, out_v, row_offset=5)
    assert got[0] is out_k and got[1] is out_v
    for t, s in ((out_k, ks), (out_v, vs)):
        want = held(s)[:, :, 5:].reshape(b * h, -1, hd)
        want = np.stack([want[u, idx[u].cpu().numpy()] for u in range(b * h)]).reshape(b, h, 11, hd)
        assert np.array_equal(f64(t), want)
    assert not big[:, :4].any() and not big[:, 15:].any()
    # attention over the same views
    q, qx = bf16(rng.standard_normal((b, h * 2, hd)))
    check_attention(q, qx, ks, vs, [42, 30])


def test_rows_that_the_store_does_not_have():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((1, 2, 9, 64))
    k, v = store_of(x, 4), store_of(x[:, :, :7], 8)
    idx = torch.tensor([[0, 8, 9, -1], [6, 7, 2**31 - 1, 3]], dtype=torch.int32, device=DEV)
    out_k, out_v = hip().mx_gather_rows(k, v, idx)
    for t, s, n in ((out_k, k, 9), (out_v, v, 7)):
        rows = held(s)[0]
        for u in range(2):
            for j, r in enumerate(idx[u].tolist()):
                assert np.array_equal(f64(t)[0, u, j], rows[u, r] if 0 <= r < n else np.zeros(64))
    only_v = hip().mx_gather_rows(None, v, idx)
    assert only_v[0] is None and torch.equal(only_v[1], out_v)
    only_k = hip().mx_gather_rows(k, None, idx[:, 1:3])
    assert only_k[1] is None and torch.equal(only_k[0], out_k[:, :, 1:3])
    assert torch.equal(hip().mx_gather_rows(k, None, idx[:1].expand(2, 4))[0][:, 0], out_k[:, 0])
    assert hip().mx_gather_rows(k, None, row_offset=9)[0].shape == (1, 2, 0, 64)
    assert not hip().mx_gather_rows(k, None, row_offset=12, n_idx=3)[0].any()


@pytest.mark.parametrize("hd,kbits,vbits", [(64, 4, 8), (128, 4, 4), (256, 8, 4)])
def test_appended_tokens(hd, kbits, vbits):
    rng = np.random.default_rng(6)
    b, h, n = 5, 3, 8
    ks, vs = (hip().MxStore(torch.full((b, h, n, hd * x // 8), 3, dtype=torch.uint8, device=DEV),
                            torch.full((b, h, n, hd // 32), 4, dtype=torch.uint8, device=DEV)) for x in (kbits, vbits))
    (k, kx), (v, vx) = bf16(keys(rng, (b, 1, h, hd))), bf16(rng.standard_normal((b, h, hd)))
    lens = [0, 7, 8, -1, 3]                                           # the third and the fourth have no such row
    at = torch.tensor(lens, dtype=torch.int32, device=DEV)
    hip().mx_append(ks, vs, k, v, at)
    assert at.tolist() == lens
    for s, x, bits in ((ks, kx[:, 0], kbits), (vs, vx, vbits)):
        codes, scale = ref.encode(x, bits)
        want_c, want_s = np.full((b, h, n, hd * bits // 8), 3), np.full((b, h, n, hd // 32), 4)
        for i, r in enumerate(lens):
            if 0 <= r < n:
                want_c[i, :, r], want_s[i, :, r] = codes[i], scale[i]
        assert np.array_equal(s.codes.cpu().numpy(), want_c) and np.array_equal(s.scale.cpu().numpy(), want_s)


# ---- attention --------------------------------------------------------------------------------------------------------

def check_attention(q, qx, ks, vs, lens, n_rows=None, n_sink=0, window=0, scale=None, **more):
    """One call against 64 bits.  Bounds: a logit's error D is that of hd + 2 roundings of fp32 sums of |q k|; a weight's is D, that
    of exp2 and of P as two bf16 numbers (2^-16), and sums of n terms add n 2^-24; the output's own rounding is 2^-8."""
    b, hq, hd = q.shape
    h = ks.shape[1]
    g = hq // h
    scale = 1 / math.sqrt(hd) if scale is None else scale
    room = min(ks.shape[2], vs.shape[2]) if n_rows is None else n_rows
    t = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse = hip().mx_attn(q, ks, vs, t, n_rows=n_rows, n_sink=n_sink, window=window, scale=scale, want_lse=True, **more)
    kx, vx = held(ks), held(vs)
    got, got_lse = f64(out), f64(lse)
    for i in range(b):
        total = room if lens is None else min(max(lens[i] + ("new_k" in more), 0), room)
        rows = ref.attended(total, n_sink, window)
        for j in range(h):
            mine = slice(j * g, (j + 1) * g)
            want, want_lse, weight, logit = ref.attention(qx[i, mine], kx[i, j, rows], vx[i, j, rows], scale)
            d = (hd + 4) * 2.0 ** -24 * logit
            rel = 2 * d + 2.0 ** -16 + 2.0 ** -21 + 2 * len(rows) * 2.0 ** -24
            tol = 2.0 ** -8 * np.abs(want) + weight * (rel * (1 + 2.0 ** -7))[:, None] + 1e-38
            assert (np.abs(got[i, mine] - want) <= tol).all(), (i, j, np.max(np.abs(got[i, mine] - want) / tol))
            fine = np.isfinite(want_lse)
            assert np.array_equal(fine, np.isfinite(got_lse[i, mine])) and (got_lse[i, mine][~fine] == -np.inf).all()
            bound = d[fine] + 2.0 ** -20 + len(rows) * 2.0 ** -24 + 4 * 2.0 ** -24 * np.abs(want_lse[fine])
            assert (np.abs(got_lse[i, mine][fine] - want_lse[fine]) <= bound).all()
    return out, lse


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kbits,vbits", [(4, 4), (8, 4), (4, 8), (8, 8)])
@pytest.mark.parametrize("group", [1, 3, 4, 7, 8, 16])
def test_attention(hd, kbits, vbits, group):
    rng = np.random.default_rng(hd + group)
    lens = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 257, 300]
    b, h, n = len(lens), 2, 300
    ks, vs = store_of(keys(rng, (b, h, n, hd)), kbits), store_of(rng.standard_normal((b, h, n, hd)), vbits)
    for s in (ks, vs):                                                # what lies behind a sequence's end must not be read
        for i, length in enumerate(lens):
            s.codes[i, :, length:], s.scale[i, :, length:] = 0xff, 0xff
    q, qx = bf16(rng.standard_normal((b, h * group, hd)))
    check_attention(q, qx, ks, vs, lens)


@pytest.mark.parametrize("hd,kbits,vbits,group,n", [(128, 4, 4, 4, 4099), (64, 8, 4, 7, 20011), (256, 4, 8, 2, 3001),
                                                    (128, 8, 8, 16, 1537), (128, 4, 4, 1, 70001)])
def test_attention_over_long_contexts(hd, kbits, vbits, group, n):
    rng = np.random.default_rng(n)
    b, h = 2, 1
    x = keys(rng, (b, h, n, hd))
    x[0, 0, n // 3] *= 4.0                                            # one row that most of the weight goes to
    ks, vs = store_of(x, kbits), store_of(rng.standard_normal((b, h, n, hd)), vbits)
    q, qx = bf16(rng.standard_normal((b, h * group, hd)))
    check_attention(q, qx, ks, vs, [n, n - 1000])
    check_attention(q, qx, ks, vs, None)
    check_attention(q, qx, ks, vs, [n, 70], n_rows=n - 5)


@pytest.mark.parametrize("n_sink,window", [(0, 1), (4, 64), (64, 200), (1, 63), (65, 129), (0, 700), (300, 299), (700, 5)])
def test_sinks_and_window(n_sink, window):
    rng = np.random.default_rng(window)
    lens = [600, 599, 0, 1, 64, 65, 130, 301]
    ks, vs = store_of(keys(rng, (8, 2, 600, 128)), 4), store_of(rng.standard_normal((8, 2, 600, 128)), 4)
    q, qx = bf16(rng.standard_normal((8, 8, 128)))
    for i, n in enumerate(lens):                                      # rows between and behind hold what must not be read
        rows = np.setdiff1d(np.arange(600), ref.attended(n, n_sink, window))
        for s in (ks, vs):
            s.codes[i, :, rows], s.scale[i, :, rows] = 0xff, 0xff
    check_attention(q, qx, ks, vs, lens, n_sink=n_sink, window=window)


def test_more_units_than_blocks():
    """One part to a unit: no workspace, the kernel writes the output itself."""
    rng = np.random.default_rng(8)
    b, h, n, hd = 300, 2, 200, 64
    ks, vs = store_of(keys(rng, (b, h, n, hd)), 4), store_of(rng.standard_normal((b, h, n, hd)), 4)
    q, qx = bf16(rng.standard_normal((b, h * 2, hd)))
    check_attention(q, qx, ks, vs, rng.integers(0, n + 1, b).tolist())


@pytest.mark.parametrize("size", [1e-30, 1e-3, 40.0, 1e4])
def test_logits_of_any_size(size):
    rng = np.random.default_rng(9)
    ks, vs = store_of(rng.standard_normal((1, 2, 500, 128)), 4), store_of(1e-3 * rng.standard_normal((1, 2, 500, 128)), 4)
    q, qx = bf16(size * rng.standard_normal((1, 8, 128)))
    check_attention(q, qx, ks, vs, [500])
    check_attention(q, qx, ks, vs, [500], scale=-0.3)
    check_attention(q, qx, ks, vs, [500], scale=0.0)


def test_rising_logits():
    """Every step's rows outweigh the last one's: the maximum moves all the time."""
    rng = np.random.default_rng(10)
    n, hd = 2048, 128
    x = rng.standard_normal((1, 1, n, hd)) * 0.1
    x[..., 0] += np.linspace(-300, 300, n)
    ks, vs = store_of(x, 8), store_of(rng.standard_normal((1, 1, n, hd)), 4)
    qx = 0.1 * rng.standard_normal((1, 4, hd))
    qx[..., 0] = np.array([3, -3, 1, 0.01])
    q, qx = bf16(qx)
    check_attention(q, qx, ks, vs, [n])


@pytest.mark.parametrize("hd,group,kbits", [(64, 4, 4), (128, 4, 8), (128, 16, 4), (256, 1, 4)])
@pytest.mark.parametrize("where", ["k", "v", "q"])
@pytest.mark.parametrize("n", [40, 3000])
def test_nan_stays_with_its_unit(hd, group, kbits, where, n):
    rng = np.random.default_rng(11)
    k, v = keys(rng, (2, 2, n, hd)), rng.standard_normal((2, 2, n, hd))
    qx = rng.standard_normal((2, 2 * group, hd))
    {"k": k, "v": v}.get(where, np.zeros((2, 2, n, hd)))[1, 0, n - 3, 5] = math.nan
    if where == "q":
        qx[1, 0, 7] = math.nan
    q, _ = bf16(qx)
    out, lse = hip().mx_attn(q, store_of(k, kbits), store_of(v, 4), want_lse=True)
    bad = torch.isnan(out).view(2, 2, group, hd)
    if where == "q":
        assert bad[1, 0, 0].all() and bad.sum() == hd
    elif where == "k":
        assert bad[1, 0].all() and bad.sum() == group * hd
    else:                                                             # a block of V is 32 columns
        assert bad[1, 0, :, :32].all() and bad.sum() == group * 32
    nan_lse = torch.isnan(lse).view(2, 2, group)
    assert nan_lse.sum() == {"q": 1, "k": group, "v": 0}[where]


@pytest.mark.parametrize("hd,kbits,vbits,group", [(64, 8, 4, 7), (128, 4, 4, 4), (256, 4, 8, 3)])
@pytest.mark.parametrize("n_sink,window", [(0, 0), (3, 70)])
def test_a_token_written_and_attended(hd, kbits, vbits, group, n_sink, window):
    rng = np.random.default_rng(12)
    lens = [0, 1, 63, 64, 65, 500, 2999, 3000, 3001, -1]              # from 3000 on there is no row for it
    b, h, n = len(lens), 2, 3000
    k, v = keys(rng, (b, h, n, hd)), rng.standard_normal((b, h, n, hd))
    (nk, nkx), (nv, nvx) = bf16(3 * rng.standard_normal((b, h, hd))), bf16(rng.standard_normal((b, h, hd)))
    q, qx = bf16(rng.standard_normal((b, h * group, hd)))
    ks, vs = store_of(k, kbits), store_of(v, vbits)
    want_k, want_v = store_of(k, kbits), store_of(v, vbits)
    at = torch.tensor(lens, dtype=torch.int32, device=DEV)
    lens = [max(x, 0) for x in lens]                                  # a negative length is none
    hip().mx_append(want_k, want_v, nk, nv, at.clamp(min=0))
    out, lse = hip().mx_attn(q, ks, vs, at, new_k=nk, new_v=nv, n_sink=n_sink, window=window, want_lse=True)
    for s, w in ((ks, want_k), (vs, want_v)):
        assert torch.equal(s.codes, w.codes) and torch.equal(s.scale, w.scale)
    after = torch.tensor([min(x + 1, n) for x in lens], dtype=torch.int32, device=DEV)
    two, two_lse = hip().mx_attn(q, want_k, want_v, after, n_sink=n_sink, window=window, want_lse=True)
    assert torch.equal(out, two) and torch.equal(lse, two_lse)
    check_attention(q, qx, want_k, want_v, after.tolist(), n_sink=n_sink, window=window)
    # n_rows ends the sequences: what has no row below it is neither written nor attended to
    ks, vs = store_of(k, kbits), store_of(v, vbits)
    out = hip().mx_attn(q, ks, vs, at, new_k=nk, new_v=nv, n_rows=64)
    want = store_of(k, kbits)
    hip().mx_append(want, store_of(v, vbits), nk, nv, torch.where(at >= 64, 10**6, at.clamp(min=0)).int())
    assert torch.equal(ks.codes, want.codes) and torch.equal(ks.scale, want.scale)
    assert torch.equal(out, hip().mx_attn(q, ks, vs, (at.clamp(min=0) + 1).clamp(max=64).int()))


def test_a_token_without_lens_takes_the_last_row():
    rng = np.random.default_rng(13)
    k, v = rng.standard_normal((1, 1, 50, 64)), rng.standard_normal((1, 1, 50, 64))
    nk, nkx = bf16(rng.standard_normal((1, 1, 64)))
    q, qx = bf16(rng.standard_normal((1, 2, 64)))
    ks, vs = store_of(k, 4), store_of(v, 4)
    hip().mx_attn(q, ks, vs, new_k=nk, new_v=nk)
    codes, scale = ref.encode(nkx, 4)
    assert np.array_equal(ks.codes.cpu().numpy()[:, :, 49], codes) and np.array_equal(vs.scale.cpu().numpy()[:, :, 49], scale)


def test_units_far_apart():
    """Offsets beyond 32 bits between the units."""
    rng = np.random.default_rng(14)
    n, hd = 600, 128
    room = torch.zeros((5 << 30,), dtype=torch.uint8, device=DEV)
    stores = []
    for i, z in enumerate((keys(rng, (2, 1, n, hd)), rng.standard_normal((2, 1, n, hd)))):
        small = store_of(z, 4)
        codes = torch.as_strided(room[i << 16:], (2, 1, n, 64), ((4 << 30) + 64, 64, 64, 1))
        scale = torch.as_strided(room[(i << 16) + (1 << 20):], (2, 1, n, 4), ((4 << 30) + 8, 4, 4, 1))
        codes.copy_(small.codes)
        scale.copy_(small.scale)
        stores.append(hip().MxStore(codes, scale))
    q, qx = bf16(rng.standard_normal((2, 4, hd)))
    check_attention(q, qx, *stores, [n, n - 1])
    back = hip().mx_gather_rows(stores[0], None)[0]
    assert np.array_equal(f64(back), held(stores[0]))
    nk, _ = bf16(rng.standard_normal((2, 1, hd)))
    hip().mx_append(*stores, nk, nk, torch.tensor([n - 1, n - 2], dtype=torch.int32, device=DEV))
    check_attention(q, qx, *stores, [n, n - 1])


def test_rows_beyond_four_gib_of_a_unit():
    """One unit of 17 million rows of 256 bytes: prompts, tokens, rows and a window at its end."""
    rng = np.random.default_rng(24)
    n, hd, last = 17 << 20, 256, 300
    s = hip().MxStore.zeros(1, 1, n, hd, 8, DEV)
    (k, kx), (v, vx) = bf16(rng.standard_normal((1, last, 1, hd))), bf16(rng.standard_normal((1, last, 1, hd)))
    other = hip().MxStore.zeros(1, 1, n, hd, 8, DEV)
    hip().mx_ingest(s, other, k, v, dst_pos=n - last)
    nk, _ = bf16(rng.standard_normal((1, 1, hd)))
    q, qx = bf16(rng.standard_normal((1, 2, hd)))
    at = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    out = hip().mx_attn(q, s, other, at, new_k=nk, new_v=nk, n_sink=3, window=last)
    back_k, back_v = hip().mx_gather_rows(s, other, row_offset=n - last)
    want = ref.decode(*ref.encode(kx[:, :last - 1].transpose(0, 2, 1, 3), 8))
    assert np.array_equal(f64(back_k)[:, :, :last - 1], want)
    token = ref.decode(*ref.encode(f64(nk), 8))
    assert np.array_equal(f64(back_k)[:, :, last - 1], token) and np.array_equal(f64(back_v)[:, :, last - 1], token)
    zeros = np.zeros((3, hd))
    want, _, weight, _ = ref.attention(qx[0], np.concatenate([zeros, f64(back_k)[0, 0]]), np.concatenate([zeros, f64(back_v)[0, 0]]), hd ** -0.5)
    assert (np.abs(f64(out)[0] - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -14 * weight).all()
    idx = torch.tensor([[n - 1, 0, n - last]], dtype=torch.int32, device=DEV)
    got = hip().mx_gather_rows(s, None, idx)[0]
    assert torch.equal(got[0, 0], torch.stack([back_k[0, 0, -1], torch.zeros_like(back_k[0, 0, 0]), back_k[0, 0, 0]]))


def test_shared_units_may_be_read():
    """A prefix that a batch shares: stride 0 over the batch."""
    rng = np.random.default_rng(15)
    one = [store_of(rng.standard_normal((1, 2, 333, 128)), 4) for _ in range(2)]
    shared = [hip().MxStore(s.codes.expand(4, -1, -1, -1), s.scale.expand(4, -1, -1, -1)) for s in one]
    q, qx = bf16(rng.standard_normal((4, 8, 128)))
    check_attention(q, qx, *shared, [333, 100, 1, 0])
    with pytest.raises(hip().DiffCacheError, match="share"):
        hip().mx_append(*shared, q[:, :2], q[:, :2], torch.zeros(4, dtype=torch.int32, device=DEV))


# ---- streams, graphs, together ----------------------------------------------------------------------------------------

def test_captured_steps_follow_the_lengths():
    """Two graphs of two caches with a workspace each, replayed in turn among eager work: every replay against an eager step."""
    rng = np.random.default_rng(16)
    b, h, g, n, hd = 2, 2, 4, 1500, 128
    k, v = keys(rng, (b, h, n, hd)), rng.standard_normal((b, h, n, hd))
    q, _ = bf16(rng.standard_normal((b, h * g, hd)))
    nk, _ = bf16(rng.standard_normal((b, h, hd)))
    nv, _ = bf16(rng.standard_normal((b, h, hd)))
    runs = []
    for start in ([700, 3], [0, 1400]):
        c = dict(ks=store_of(k, 4), vs=store_of(v, 4), lens=torch.tensor(start, dtype=torch.int32, device=DEV),
                 ws=torch.empty(hip().mx_attn_workspace_bytes(b * h, g, hd, n), dtype=torch.uint8, device=DEV),
                 out=torch.empty_like(q), lse=torch.empty((b, h * g), device=DEV), start=start)
        c["eager"] = (store_of(k, 4), store_of(v, 4))

        def step(c=c):
            hip().mx_attn(q, c["ks"], c["vs"], c["lens"], new_k=nk, new_v=nv, out=c["out"], lse=c["lse"], workspace=c["ws"])
            c["lens"].add_(1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        c["lens"].copy_(torch.tensor(start, dtype=torch.int32))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        c["graph"] = graph
        runs.append(c)
    for i in range(6):
        for c in runs:
            for t in (q, nk, nv):
                t.copy_(torch.randn(t.shape, device=DEV))
            c["graph"].replay()
            lens = torch.tensor([x + i for x in c["start"]], dtype=torch.int32, device=DEV)
            out, lse = hip().mx_attn(q, *c["eager"], lens, new_k=nk, new_v=nv, want_lse=True)
            if i % 2:
                torch.cuda.synchronize()
            assert torch.equal(c["out"], out) and torch.equal(c["lse"], lse), i
            assert torch.equal(c["ks"].codes, c["eager"][0].codes) and torch.equal(c["lens"], lens + 1)


def test_writing_and_reading_back_captured():
    """Prompts, a token and rows read back in one graph, replayed on other inputs among eager work: every replay against eager calls."""
    b, h, seq, hd = 2, 3, 150, 128
    src = [torch.zeros((b, seq, h, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    new = [torch.zeros((b, h, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    lens = torch.tensor([seq, 20], dtype=torch.int32, device=DEV)
    idx = torch.zeros((b * h, 9), dtype=torch.int32, device=DEV)
    stores = [[m.zeros(b, h, seq + 1, hd, bits, DEV) for bits in (4, 8)] for m in (hip().MxStore, hip().MxStore)]

    def work(k, v):
        hip().mx_ingest(k, v, *src, lens=lens)
        hip().mx_append(k, v, *new, lens)
        return hip().mx_gather_rows(k, v) + hip().mx_gather_rows(k, v, idx, row_offset=1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured = work(*stores[0])
    for i in range(5):
        for t in src + new:
            t.copy_(torch.randn(t.shape, device=DEV) * 2.0 ** (10 * i - 20))
        lens.copy_(torch.tensor([seq - i, 20 + 25 * i], dtype=torch.int32))
        idx.copy_(torch.randint(0, seq, idx.shape, device=DEV))
        graph.replay()
        eager = work(*stores[1])
        if i % 2:
            torch.cuda.synchronize()
        for x, y in zip(captured, eager):
            assert torch.equal(x, y), i
        for x, y in zip(*stores):
            assert torch.equal(x.codes, y.codes) and torch.equal(x.scale, y.scale)


def test_two_streams_at_once():
    rng = np.random.default_rng(17)
    ks, vs = store_of(keys(rng, (2, 4, 9000, 128)), 4), store_of(rng.standard_normal((2, 4, 9000, 128)), 4)
    qs = [bf16(rng.standard_normal((2, 16, 128)))[0] for _ in range(2)]
    want = [hip().mx_attn(q, ks, vs) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(hip().mx_attn(qs[i], ks, vs))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_a_run_of_all_of_them():
    """Prompts in, tokens written and attended, rows read back: the bf16 rows under the framework's gathered attention give the
    same attention."""
    rng = np.random.default_rng(18)
    b, h, g, hd, seq, steps = 2, 2, 4, 128, 205, 4
    prompt = [4, seq]
    (k, kx), (v, vx) = bf16(keys(rng, (b, seq, h, hd))), bf16(rng.standard_normal((b, seq, h, hd)))
    ks, vs = (hip().MxStore.zeros(b, h, seq + steps, hd, bits, DEV) for bits in (8, 4))
    lens = torch.tensor(prompt, dtype=torch.int32, device=DEV)
    hip().mx_ingest(ks, vs, k, v, lens=lens)
    for i in range(steps):
        nk, nv = bf16(rng.standard_normal((b, h, hd)))[0], bf16(rng.standard_normal((b, h, hd)))[0]
        q, qx = bf16(rng.standard_normal((b, h * g, hd)))
        out = hip().mx_attn(q, ks, vs, lens, new_k=nk, new_v=nv)
        lens += 1
        check_attention(q, qx, ks, vs, lens.tolist())
        bk, bv = hip().mx_gather_rows(ks, vs)
        for s in range(b):
            n = prompt[s] + i + 1
            same = hip().gather_attn(q[s:s + 1], bk[s:s + 1], bv[s:s + 1], None, 0, 0, 0, 0, n)
            # both round to bf16 what is within a few 2^-16 of the same number
            assert (f64(same)[0] - f64(out)[s]).__abs__().max() <= 2.0 ** -7 * max(1.0, np.abs(f64(out)[s]).max())


def test_sizes_of_nothing():
    s = hip().MxStore.zeros(1, 2, 5, 64, 4, DEV)
    x = torch.zeros((1, 0, 2, 64), dtype=torch.bfloat16, device=DEV)
    hip().mx_ingest(s, s, x, x)
    q = torch.ones((1, 4, 64), dtype=torch.bfloat16, device=DEV)
    out, lse = hip().mx_attn(q, s, s, n_rows=0, want_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    empty = hip().MxStore.zeros(1, 2, 0, 64, 4, DEV)
    out, lse = hip().mx_attn(q, empty, empty, want_lse=True)
    assert not out.any() and (lse == -math.inf).all()
    none = hip().MxStore.zeros(0, 2, 5, 64, 4, DEV)
    assert hip().mx_attn(q[:0], none, none).shape[0] == 0
    assert hip().mx_gather_rows(none, none)[0].shape == (0, 2, 5, 64)


def test_arguments_in_other_forms():
    """q as one row a sequence, strided, off its alignment and as the output; stores of unequal room; out and lse given."""
    rng = np.random.default_rng(25)
    b, h, g, hd, n = 3, 2, 4, 128, 700
    ks, vs = store_of(keys(rng, (b, h, n, hd)), 4), store_of(rng.standard_normal((b, h, n + 9, hd)), 8)
    q, qx = bf16(rng.standard_normal((b, h * g, hd)))
    want, want_lse = check_attention(q, qx, ks, vs, [700, 650, 1])
    lens = torch.tensor([700, 650, 1], dtype=torch.int32, device=DEV)
    assert torch.equal(hip().mx_attn(q.view(b, 1, h * g * hd), ks, vs, lens), want)
    wide = torch.zeros((b, h * g, 2 * hd + 1), dtype=torch.bfloat16, device=DEV)
    wide[..., 1:hd + 1] = q
    assert torch.equal(hip().mx_attn(wide[..., 1:hd + 1], ks, vs, lens), want)
    flat = torch.zeros(q.numel() + 3, dtype=torch.bfloat16, device=DEV)
    flat[3:] = q.flatten()
    assert torch.equal(hip().mx_attn(flat[3:].view(q.shape), ks, vs, lens), want)
    lse = torch.empty((b, h * g), device=DEV)
    same = q.clone()
    out, got = hip().mx_attn(same, ks, vs, lens, out=same, lse=lse)
    assert out is same and got is lse and torch.equal(out, want) and torch.equal(lse, want_lse)
    ws = torch.full((hip().mx_attn_workspace_bytes(b * h * 7, g, hd, 9 * n),), 0xff, dtype=torch.uint8, device=DEV)
    long_k, long_v = store_of(keys(rng, (b, h, 5000, hd)), 4), store_of(rng.standard_normal((b, h, 5000, hd)), 4)
    check_attention(q, qx, long_k, long_v, [4999, 3, 0], workspace=ws)          # whatever it held, and more of it than needed
    check_attention(q, qx, long_k, long_v, [0, 0, 0], workspace=ws)
    # the token's rows in the shape of a model's projection, cut out of it
    fused = torch.randn((b, 1, 3 * h, hd), device=DEV).to(torch.bfloat16)
    nk, nv = fused[:, :, h:2 * h], fused[:, :, 2 * h:]
    one, two = store_of(held(ks)[:, :, :650], 4, 701), store_of(held(vs)[:, :, :650], 8, 701)
    hip().mx_attn(q, one, two, lens.clamp(max=650), new_k=nk, new_v=nv)
    back_k, back_v = hip().mx_gather_rows(one, two, lens.clamp(max=650).view(b, 1).expand(b, h).reshape(b * h, 1))
    for got, new, bits in ((back_k, nk, 4), (back_v, nv, 8)):
        assert np.array_equal(f64(got)[:, :, 0], ref.decode(*ref.encode(f64(new)[:, 0], bits)))


def test_very_many_sequences():
    rng = np.random.default_rng(26)
    b, n, hd = 70001, 2, 64
    x = np.zeros((b, 1, n, hd))
    x[:, 0, :, :4] = rng.integers(-6, 7, (b, n, 4)) / 2
    x[:, 0, :, 32] = 6
    ks = vs = store_of(x, 4)
    q = torch.zeros((b, 2, hd), dtype=torch.bfloat16, device=DEV)
    q[:, :, 0] = 1
    lens = torch.arange(b, dtype=torch.int32, device=DEV) % 3
    out, lse = hip().mx_attn(q, ks, vs, lens, scale=1.0, want_lse=True)
    live = np.arange(n)[None] < (np.arange(b) % 3)[:, None]
    e = np.where(live, np.exp(held(ks)[:, 0, :, 0]), 0.0)
    total = e.sum(1)
    want = np.where(total[:, None] > 0, (e[:, :, None] * held(vs)[:, 0]).sum(1) / np.maximum(total, 1e-30)[:, None], 0.0)
    assert (np.abs(f64(out) - want[:, None]) <= 2.0 ** -8 * np.abs(want)[:, None] + 2.0 ** -13 * 6).all()
    assert np.array_equal(np.isinf(f64(lse)[:, 0]), total == 0)


def test_wrappers_refuse_on_the_gpu():
    m = hip()
    ks, vs = m.MxStore.zeros(2, 2, 40, 128, 4, DEV), m.MxStore.zeros(2, 2, 40, 128, 8, DEV)
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=DEV)
    nk = torch.zeros((2, 2, 128), dtype=torch.bfloat16, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    src = torch.zeros((2, 10, 2, 128), dtype=torch.bfloat16, device=DEV)
    bad = [
        (lambda: m.mx_attn(q.half(), ks, vs, lens), "bf16"), (lambda: m.mx_attn(q[:, :7], ks, vs, lens), "values"),
        (lambda: m.mx_attn(q.cpu(), ks, vs, lens), "GPU memory"), (lambda: m.mx_attn(q, ks, vs, lens.long()), "int32"),
        (lambda: m.mx_attn(q, ks, vs, lens[:1]), "2 elements"), (lambda: m.mx_attn(q, ks, vs, lens.cpu()), "GPU memory"),
        (lambda: m.mx_attn(q, ks, vs, lens, n_rows=41), "outside"), (lambda: m.mx_attn(q, ks, vs, lens, window=-1), "negative"),
        (lambda: m.mx_attn(q, ks, vs, lens, new_k=nk), "together"), (lambda: m.mx_attn(q, ks, vs, lens, new_k=nk, new_v=nk[:1]), "new_v"),
        (lambda: m.mx_attn(q, ks, vs, lens, out=q.float()), "out"), (lambda: m.mx_attn(q, ks, vs, lens, out=q[:, :4]), "out"),
        (lambda: m.mx_attn(q, ks, vs, lens, lse=q.float()), "lse"), (lambda: m.mx_attn(q.repeat(1, 5, 1), ks, vs, lens), "group"),
        (lambda: m.mx_attn(q, ks, m.MxStore.zeros(2, 1, 40, 128, 4, DEV), lens), "belong"),
        (lambda: m.mx_attn(q, ks, m.MxStore.zeros(2, 2, 40, 64, 4, DEV), lens), "belong"),
        (lambda: m.mx_ingest(ks, vs, src, src, dst_pos=31), "outside"), (lambda: m.mx_ingest(ks, vs, src, src[:, :9]), "v_src"),
        (lambda: m.mx_ingest(ks, vs, src.float(), src), "k_src"), (lambda: m.mx_ingest(ks, vs, src[0], src[0]), "k_src"),
        (lambda: m.mx_ingest(ks, vs, src, src, dst_pos=-1), "outside"), (lambda: m.mx_ingest(ks, vs, src, src, lens=lens.float()), "int32"),
        (lambda: m.mx_append(ks, vs, nk, nk[:, :1], lens), "new_v"), (lambda: m.mx_append(ks, vs, nk, nk, None), "null"),
        (lambda: m.mx_gather_rows(None, None), "neither"), (lambda: m.mx_gather_rows(ks, vs, lens), "idx"),
        (lambda: m.mx_gather_rows(ks, vs, lens.view(1, 2).expand(4, 2), n_idx=3), "idx"),
        (lambda: m.mx_gather_rows(ks, vs, torch.zeros((4, 2), device=DEV)), "idx"), (lambda: m.mx_gather_rows(ks, vs, row_offset=-1), "negative"),
        (lambda: m.mx_gather_rows(ks, vs, n_idx=10, out_k=nk.view(2, 2, 1, 128)), "out_k"),
        (lambda: m.mx_gather_rows(ks, None, n_idx=1, out_v=nk.view(2, 2, 1, 128)), "each with its store"),
        (lambda: m.mx_gather_rows(ks, vs, n_idx=5, out_k=src[:, :5].transpose(1, 2)), "share"),
        (lambda: m.MxStore(ks.codes, vs.scale.cpu()), "GPU memory"),
    ]
    before = ks.codes.clone()
    for call, message in bad:
        with pytest.raises(m.DiffCacheError, match=message):
            call()
    small = torch.empty(256, dtype=torch.uint8, device=DEV)
    big = [m.MxStore.zeros(2, 2, 5000, 128, 4, DEV) for _ in range(2)]
    with pytest.raises(m.DiffCacheError, match="needed"):
        m.mx_attn(q, *big, lens, workspace=small)
    assert torch.equal(ks.codes, before) and not torch.isnan(m.mx_attn(q, ks, vs, lens).float()).any()
