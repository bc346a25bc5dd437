"""Tokens written into pages (dc_paged_append_bf16) against 64 bits."""
import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def near(got, want, mag):
    """The result's own rounding (2^-8 of it); sine and cosine 1.2e-7 each and three fp32 operations, of the pair's magnitude."""
    err = (got.double() - want).abs()
    assert (err <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * mag).all(), err.max()


@pytest.mark.parametrize("hd,rot,interleaved", [(64, 64, False), (128, 128, False), (128, 32, False), (256, 256, False), (256, 64, True), (128, 128, True),
                                                (64, 16, True), (64, 48, False), (128, 0, False)])
@pytest.mark.parametrize("form", ["one", "padded", "packed"])
def test_rows_and_queries(hd, rot, interleaved, form):
    from diffcache_amd import _hip as hip
    g = torch.Generator(device=DEV).manual_seed(hd + rot)
    h, hq, page, n_pages = 2, 6, 16, 40
    starts = [0, 15, 200]
    counts = {"one": [1, 1, 1], "padded": [0, 37, 21], "packed": [5, 0, 60]}[form]
    b = 3
    table = torch.randperm(n_pages, generator=g, device=DEV)[:3 * 13].to(torch.int32).view(3, 13)     # rows up to 207
    table[2, 12] = -1 if form == "padded" else n_pages
    lead = {"one": (3,), "padded": (3, 37), "packed": (70,)}[form]
    x = torch.randn((*lead, (hq + 2 * h) * hd), generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = (t.unflatten(-1, (-1, hd)) for t in x.split([hq * hd, h * hd, h * hd], -1))
    kp, vp = (torch.randn((n_pages, h, page, hd), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
    want_k, want_v = kp.double(), vp.double()
    cu = [2, 7, 7, 67] if form == "packed" else None
    inv = (1e6 ** (-torch.arange(rot // 2, device=DEV) / max(rot // 2, 1))).float() if rot else None
    span = ref.spans(3, starts, cu, counts if form == "padded" else None, {"one": 1, "padded": 37, "packed": 60}[form], 70)
    assert [c for _, c, _ in span] == counts
    q_out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=DEV) if rot else None
    got = hip.paged_append(kp, vp, table, k, v, i32(starts), cu=None if cu is None else i32(cu),
                           counts=i32(counts) if form == "padded" else None, max_new=60 if form == "packed" else None,
                           q=q if rot else None, q_out=q_out, inv_freq=inv, interleaved=interleaved)
    assert got is q_out
    flat = [t.reshape(-1, t.shape[-2], hd) for t in (q, k, v)]
    mag_k = torch.zeros_like(want_k)
    untouched = torch.ones(flat[0].shape[0], dtype=torch.bool, device=DEV)
    for s, (first, count, start) in enumerate(span):
        if count == 0:
            continue
        pos = torch.arange(start, start + count, device=DEV)[:, None]
        mine = slice(first, first + count)
        tq, tk = (ref.rotate(t[mine], pos, inv, interleaved) if rot else t[mine].double() for t in flat[:2])
        untouched[mine] = False
        for i in range(count):
            at = ref.place(table[s].tolist(), start + i, page, n_pages)
            if at is not None:
                want_k[at[0], :, at[1]], want_v[at[0], :, at[1]] = tk[i], flat[2][first + i].double()
                mag_k[at[0], :, at[1]] = tk[i].abs().amax(-1, keepdim=True)
        if rot:
            near(q_out.view(-1, hq, hd)[mine], tq, tq.abs().amax(-1, keepdim=True))
    near(kp, want_k, mag_k)
    assert torch.equal(vp.double(), want_v)
    if rot:
        assert (q_out.view(-1, hq, hd)[untouched] == 7).all()


@pytest.mark.parametrize("sections", [(16, 24, 24), (64,), (0, 30, 1, 33), (10, 54)])
def test_positions_of_several_axes(sections):
    from diffcache_amd import _hip as hip
    g = torch.Generator(device=DEV).manual_seed(3)
    b, t, h, hd, page = 2, 300, 3, 128, 32
    kp, vp = (torch.zeros((24, h, page, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = torch.arange(24, dtype=torch.int32, device=DEV).view(2, 12)
    k, v, q = (torch.randn((b, t, n, hd), generator=g, device=DEV).to(torch.bfloat16) for n in (h, h, 5))
    pos = torch.randint(-50, 1 << 20, (b, t, len(sections)), generator=g, device=DEV).to(torch.int32)
    inv = (500000.0 ** (-torch.arange(64, device=DEV) / 64)).float()
    out = hip.paged_append(kp, vp, table, k, v, q=q, inv_freq=inv, pos=pos, sections=sections)
    for i in range(b):
        tq, tk = (ref.rotate(x[i], pos[i], inv, sections=sections) for x in (q, k))
        near(out[i], tq, tq.abs().amax(-1, keepdim=True))
        rows = kp[table[i].long()].permute(0, 2, 1, 3).flatten(0, 1)[:t]
        near(rows, tk, tk.abs().amax(-1, keepdim=True))
