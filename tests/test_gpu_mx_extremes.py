"""Attention over the block-scaled cache where logits leave fp32's range: they are the infinities that the formula in fp32 gives."""
import math

import numpy as np
import pytest
import torch

from oracle import mx as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BIG = 2.0 ** 124                           # held exactly in 4 and in 8 bits; 16 of them are beyond fp32


def hip():
    from diffcache_amd import _hip
    return _hip


def store_of(x, bits):
    codes, scale = ref.encode(x, bits)
    return hip().MxStore(torch.from_numpy(codes).to(DEV), torch.from_numpy(scale).to(DEV))


def case(n, hd, bits, group, low, seed=0):
    """Keys whose rows `low` give every head but the last logits of -16 BIG and the last -1; the others' logits are small whole
    numbers over 8.  Values are numbers of the 4-bit format: all of it is exact up to the weights."""
    rng = np.random.default_rng(seed)
    k, v = np.zeros((1, 1, n, hd)), rng.choice([-6.0, -4, -3, -2, -1, 0, 1, 2, 3, 4, 6], (1, 1, n, hd))
    k[..., 0] = rng.integers(-4, 5, n)
    k[0, 0, low, hd - 1] = -BIG            # (a block of its own)
    q = np.zeros((1, group, hd))
    q[..., 0], q[..., hd - 1] = 1 / 8, 16
    q[0, -1, hd - 1] = 1 / BIG
    return torch.from_numpy(q).to(torch.bfloat16).to(DEV), q, store_of(k, bits), store_of(v, 4), k[0, 0], v[0, 0]


def check(out, lse, q, k, v):
    """Logits are exact in fp32, exp2 and the sums of n weights are off by (4 + n) 2^-23 and P by 2^-16 of a weight, the output by
    its own rounding."""
    n = len(k)
    for i, (o, e) in enumerate(zip(out.double().cpu().numpy()[0], lse.double().cpu().numpy()[0])):
        x = q[0, i] @ k.T
        x = np.where(x < -3.4e38, -np.inf, x)
        live = x > -np.inf
        if not live.any():
            assert not o.any() and e == -np.inf
            continue
        p = np.where(live, np.exp(x - x[live].max()), 0.0)
        want, weight = p @ v / p.sum(), p @ np.abs(v) / p.sum()
        rel = 2.0 ** -15 + (4 + n) * 2.0 ** -23
        assert (np.abs(o - want) <= 2.0 ** -8 * np.abs(want) + weight * rel * (1 + 2.0 ** -7)).all(), i
        assert abs(e - (x[live].max() + math.log(p.sum()))) <= rel + 2.0 ** -20


LOW = {
    "the first rows": lambda n: np.arange(n) < min(n // 2, 700),
    "all but the last row": lambda n: np.arange(n) < n - 1,
    "all but the first row": lambda n: np.arange(n) > 0,
    "every other run of 64": lambda n: np.arange(n) // 64 % 2 == 0,
    "all rows": lambda n: np.arange(n) >= 0,
}


@pytest.mark.parametrize("low", list(LOW))
@pytest.mark.parametrize("n", [1, 50, 700, 5000])
@pytest.mark.parametrize("hd,bits,group", [(64, 4, 4), (128, 8, 7), (128, 4, 16), (256, 4, 2)])
def test_logits_below_fp32(hd, bits, group, n, low):
    q_t, q, ks, vs, k, v = case(n, hd, bits, group, LOW[low](n))
    out, lse = hip().mx_attn(q_t, ks, vs, scale=1.0, want_lse=True)
    check(out, lse, q, k, v)


def test_a_token_behind_rows_below_fp32():
    n = 900
    q_t, q, ks, vs, k, v = case(n, 128, 4, 4, np.arange(n) >= 0)
    k[-1, 127] = 0
    new_k, new_v = (torch.from_numpy(x[-1:][None]).to(torch.bfloat16).to(DEV) for x in (k, v))
    lens = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    out, lse = hip().mx_attn(q_t, ks, vs, lens, new_k=new_k, new_v=new_v, scale=1.0, want_lse=True)
    check(out, lse, q, k, v)


@pytest.mark.parametrize("n", [40, 5000])
def test_a_nan_in_a_value_of_weight_zero(n):
    """0 NaN is NaN: an attended row's NaN reaches the outputs of its 32 columns whatever its weight, as in the formula."""
    q_t, q, ks, vs, k, v = case(n, 128, 4, 4, np.arange(n) < n - 5)
    v = v[None, None].copy()
    v[0, 0, 3, 40] = math.nan
    out, lse = hip().mx_attn(q_t, ks, store_of(v, 4), scale=1.0, want_lse=True)
    bad = torch.isnan(out[0])
    assert bad[:, 32:64].all() and bad.sum() == 4 * 32 and not torch.isnan(lse).any()
    # all rows of weight zero, and that one
    q_t, q, ks, vs, k, v = case(n, 128, 4, 4, np.arange(n) >= 0)
    v = v[None, None].copy()
    v[0, 0, 3, 40] = math.nan
    out, lse = hip().mx_attn(q_t, ks, store_of(v, 4), scale=1.0, want_lse=True)
    bad = torch.isnan(out[0])
    assert bad[:, 32:64].all() and bad.sum() == 4 * 32
    assert (lse[0, :3] == -math.inf).all() and torch.isfinite(lse[0, 3])


@pytest.mark.parametrize("n", [40, 5000])
def test_logits_above_fp32(n):
    """A logit of +inf leaves no weights that are numbers: NaN, for its head alone."""
    q_t, q, ks, vs, k, v = case(n, 128, 4, 4, np.arange(n) == n - 2)
    q_t = q_t.clone()
    q_t[0, 1] = -q_t[0, 1]
    out, lse = hip().mx_attn(q_t, ks, vs, scale=1.0, want_lse=True)
    bad = torch.isnan(out[0])
    assert bad[1].all() and bad.sum() == 128
    assert torch.isnan(lse[0, 1]) and torch.isfinite(lse[0, [0, 2, 3]]).all()


def test_eight_million_sequences():
    """Units of eight waves would be more threads than a launch takes: they are of four."""
    b, n, hd = 1 << 23, 257, 64
    rng = np.random.default_rng(3)
    k, v = rng.integers(-2, 3, (1, 1, n, hd)) / 2, rng.choice([-6.0, -3, -1, 0, 1, 2, 4], (1, 1, n, hd))
    m = hip()
    ks, vs = (m.MxStore(s.codes.expand(b, -1, -1, -1), s.scale.expand(b, -1, -1, -1)) for s in (store_of(k, 4), store_of(v, 4)))
    q = torch.from_numpy(rng.integers(-4, 5, (1, 1, hd)) / 4).to(torch.bfloat16).to(DEV)
    lens = torch.arange(b, dtype=torch.int32, device=DEV) % (n + 1)
    out, lse = m.mx_attn(q.expand(b, 1, hd), ks, vs, lens, scale=0.125, want_lse=True)
    qx = q.double().cpu().numpy()[0]
    want = [ref.attention(qx, k[0, 0, :i], v[0, 0, :i], 0.125) for i in range(n + 1)]
    # logits are exact; weights, their sums and P as in check()
    rel = 2.0 ** -15 + (4 + n) * 2.0 ** -23
    o = torch.from_numpy(np.concatenate([x[0] for x in want])).to(DEV)
    tol = 2.0 ** -8 * o.abs() + torch.from_numpy(np.concatenate([x[2] for x in want])).to(DEV) * rel * (1 + 2.0 ** -7)
    e = torch.from_numpy(np.concatenate([x[1] for x in want])).to(DEV)
    for lo in range(0, b, 1 << 20):
        at = lens[lo:lo + (1 << 20)].long()
        assert ((out[lo:lo + (1 << 20), 0].double() - o[at]).abs() <= tol[at]).all()
        got = lse[lo:lo + (1 << 20), 0].double()
        assert (got[at == 0] == -math.inf).all() and ((got - e[at])[at > 0].abs() <= rel + 2.0 ** -20).all()
