"""Attention over pages (dc_paged_attn_bf16) against 64 bits: one token and many, every layout of tokens, windows, missing pages."""
import math

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bf(shape, g, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(torch.bfloat16)


def build(b, h, hd, page, lengths, seed=0, spare=2):
    """Pages in any order, with rows of NaN where no sequence has any, and the table."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    wide = max(1, max((n + page - 1) // page for n in lengths))
    n_pages = sum((n + page - 1) // page for n in lengths) + spare
    k, v = (torch.full((n_pages, h, page, hd), math.nan, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.full((b, wide), -1, dtype=torch.int32, device=DEV)
    order = torch.randperm(n_pages, generator=g, device=DEV).tolist()
    for i, n in enumerate(lengths):
        for j in range((n + page - 1) // page):
            at = order.pop()
            table[i, j] = at
            m = min(page, n - j * page)
            k[at, :, :m], v[at, :, :m] = bf((h, m, hd), g), bf((h, m, hd), g)
    return k, v, table, g


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def check(got, lse, want, p_bits, hd):
    """got, lse against oracle.attend's; p_bits: what a weight may lose when it is rounded.

    The output's own rounding is 2^-8 of it at most.  A weight's relative error: p_bits, and that of its logit: hd products summed in
    fp32 are off by at most hd 2^-24 of the sum of their magnitudes, with queries and keys of standard normal numbers 0.64 sqrt(hd)
    after the scale: 256 * 2^-24 * 10.2 = 1.6e-4 at 256 columns (times two for sums over all rows)."""
    out, want_lse, weight = want
    live = ~out.isnan().any(-1).any(-1)
    err = (got.double() - out).abs()[live]
    bound = (2.0 ** -8 * out.abs() + (p_bits + 2.0 ** -11.5) * weight)[live]
    assert (err <= bound).all(), (err / bound).max()
    # and all of it together well below that: rounding errors are independent of each other
    assert err.square().sum().sqrt() <= 3e-3 * out[live].square().sum().sqrt() + 1e-30
    e = (lse.double() - want_lse)[live]
    e = e[want_lse[live].isfinite()]
    assert torch.equal(lse[live].isfinite(), want_lse[live].isfinite())
    assert e.numel() == 0 or e.abs().max() <= 4e-4



@pytest.mark.parametrize("hd,page,h,group", [(64, 16, 2, 1), (128, 16, 2, 4), (128, 64, 1, 7), (256, 32, 2, 4), (64, 256, 1, 16), (256, 16, 1, 16),
                                             (128, 32, 3, 5), (128, 4096, 2, 2)])
@pytest.mark.parametrize("lengths", [[1], [2, 17, 64], [33, 1, 300], [1100, 513], [5000]])
def test_one_token(hd, page, h, group, lengths):
    from diffcache_amd import _hip as hip
    b = len(lengths)
    k, v, table, g = build(b, h, hd, page, lengths, seed=hd + page)
    q = bf((b, h * group, hd), g)
    out, lse = hip.paged_attn(q, k, v, table, i32([n - 1 for n in lengths]), want_lse=True)
    want = ref.attend(q, k, v, table, [(i, 1, n - 1) for i, n in enumerate(lengths)], table.shape[1] * page, hd ** -0.5)
    check(out, lse, want, 2.0 ** -15, hd)


@pytest.mark.parametrize("hd,page,h,group", [(64, 16, 2, 2), (128, 64, 2, 4), (256, 32, 1, 3)])
@pytest.mark.parametrize("tokens,starts", [(3, [0, 40, 200]), (4, [61, 0, 1500]), (40, [0, 5, 130]), (150, [0, 700, 64])])
def test_several_tokens(hd, page, h, group, tokens, starts):
    from diffcache_amd import _hip as hip
    b, lengths = len(starts), [s + tokens for s in starts]
    k, v, table, g = build(b, h, hd, page, lengths, seed=tokens)
    q = bf((b, tokens, h * group, hd), g)
    out, lse = hip.paged_attn(q, k, v, table, i32(starts), want_lse=True)
    want = ref.attend(q.flatten(0, 1), k, v, table, [(i * tokens, tokens, s) for i, s in enumerate(starts)], table.shape[1] * page, hd ** -0.5)
    check(out.flatten(0, 1), lse.flatten(0, 1), want, 2.0 ** -15 if tokens * group <= 16 else 2.0 ** -8, hd)
