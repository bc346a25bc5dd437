"""Attention over pages at the ends of what its arguments may be."""
import pytest
import torch

from test_gpu_paged_attn import DEV, build, i32

pytestmark = pytest.mark.gpu

NEW = [1, 3, 50]       # one token, a few in the registers' kernel, tiles through LDS


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_the_largest_scale(hd, new):
    """Logits are products first: those of queries of 0 are 0 under any scale, and small ones come back into range."""
    from diffcache_amd import _hip as hip
    h, group, page, n = 2, 2, 32, 300
    k, v, table, g = build(1, h, hd, page, [n + new], 31)
    q = torch.zeros((1, new, h * group, hd), dtype=torch.bfloat16, device=DEV)
    q[..., 1::2, 5] = 2.0 ** -20               # (the other heads' logits are 0)
    k[..., 5] = torch.randint(0, 8, k.shape[:3], generator=g, device=DEV).to(torch.bfloat16)
    small = k.clone()
    small[..., 5] *= 2.0 ** -105               # products of 2^-125 times 0 to 7: exact, and none below fp32's normal numbers
    scale = 2.0 ** 127 * 1.375                 # 2.34e38
    out, lse = hip.paged_attn(q, small, v, table, i32([n]), scale=scale, want_lse=True)
    # the same logits to the bit
    want = hip.paged_attn(q * 2.0 ** 20, k, v, table, i32([n]), scale=5.5, want_lse=True)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1]) and out.isfinite().all() and lse.isfinite().all()
    with pytest.raises(hip.DiffCacheError, match="scale"):
        hip.paged_attn(q, k, v, table, i32([n]), scale=2.4e38)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf")])
@pytest.mark.parametrize("low", [3, 100, 348, 399])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", NEW)
def test_an_infinity_whose_weight_is_below_fp32(new, hd, low, bad):
    """An infinity in V of a row whose weight, exp(-1600), fp32 does not hold: its column is that infinity or NaN (which one goes by the steps' order),
    never a number, and the other columns know nothing of it."""
    from diffcache_amd import _hip as hip
    n, page = 400, 16
    k, v, table, g = build(1, 1, hd, page, [n + new], 33)
    k[..., 1:], k[..., 0] = 0, 8
    k[int(table[0, low // page]), 0, low % page, 0] = -8
    q = torch.zeros((1, new, 2, hd), dtype=torch.bfloat16, device=DEV)
    q[..., 0] = 100
    clean = hip.paged_attn(q, k, v, table, i32([n]), scale=1.0, want_lse=True)
    v[int(table[0, low // page]), 0, low % page, 7] = bad
    out, lse = hip.paged_attn(q, k, v, table, i32([n]), scale=1.0, want_lse=True)
    assert ((out[..., 7] == bad) | out[..., 7].isnan()).all()
    rest = [c for c in range(hd) if c != 7]
    assert torch.equal(out[..., rest], clean[0][..., rest]) and torch.equal(lse, clean[1]) and out[..., rest].isfinite().all()
