"""Pages where it can go wrong: nothing to attend to, numbers that are not finite, ids that are no page's, long offsets, other layouts,
streams, graphs, and the same call twice."""
import math

import pytest
import torch

from oracle import paged as ref
from test_gpu_paged_attn import DEV, bf, build, check, i32

pytestmark = pytest.mark.gpu

NEW = [1, 3, 50]       # one token, a few in the registers' kernel, tiles through LDS


def tokens_of(b, new, h, group, hd, g):
    return bf((b, new, h * group, hd), g)


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_nothing_to_attend_to(hd, new):
    from diffcache_amd import _hip as hip
    k, v, table, g = build(3, 2, hd, 16, [100 + new, 100 + new, 900 + new], 1)
    table[0] = -1                              # no page at all
    table[1, :] = k.shape[0]                   # ids behind the last page
    table[2, 20:] = 2 ** 31 - 1                # only the first 320 rows have one
    q = tokens_of(3, new, 2, 2, hd, g)
    out, lse = hip.paged_attn(q, k, v, table, i32([100, 100, 900]), want_lse=True)
    assert (out[:2] == 0).all() and (lse[:2] == -math.inf).all()
    want = ref.attend(q.flatten(0, 1), k, v, table, [(0, 0, 0), (0, 0, 0), (2 * new, new, 900)], table.shape[1] * 16, hd ** -0.5)
    check(out.flatten(0, 1), lse.flatten(0, 1), want, 2.0 ** -8, hd)
    # a window of which no row has a page
    out, lse = hip.paged_attn(q[2:], k, v, table[2:], i32([900]), window=64, want_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("new", NEW)
def test_lengths_that_are_none(new):
    """No tokens, starts below zero and beyond the rows, and a call of no sequences."""
    from diffcache_amd import _hip as hip
    h, group, hd = 2, 2, 64
    k, v, table, g = build(4, h, hd, 16, [40 + new] * 4, 2)
    k.nan_to_num_(0.5), v.nan_to_num_(0.25)
    q = tokens_of(4, new, h, group, hd, g)
    out, lse = torch.full_like(q, 2.0), torch.full(q.shape[:3], 5.0, device=DEV)
    counts, starts = [0, new, -3, 10 ** 6], [40, -7, 40, 2 ** 31 - 1]
    hip.paged_attn(q, k, v, table, i32(starts), counts=i32(counts), n_rows=30, out=out, lse=lse)
    span = ref.spans(4, starts, None, counts, new, 4 * new)
    assert [c for _, c, _ in span] == [0, new, 0, new]
    # (a token far beyond the rows attends to all of them; its row number is only that of the window)
    span[3] = (span[3][0], new, 10 ** 6)
    want = ref.attend(q.flatten(0, 1), k, v, table, span, 30, hd ** -0.5)
    check(out.flatten(0, 1), lse.flatten(0, 1), want, 2.0 ** -8, hd)
    assert (out[0] == 2).all() and (out[2] == 2).all() and (lse[0] == 5).all() and (lse[2] == 5).all()
    none = hip.paged_attn(q[:0], k, v, table[:0], i32([]))
    assert none.shape == (0, new, h * group, hd)
    assert hip.paged_attn(q[:, :0], k, v, table, i32(starts)).numel() == 0
    empty, cu = q.flatten(0, 1)[:0], i32([0] * 5)
    assert hip.paged_attn(empty, k, v, table, i32(starts), cu=cu, max_new=7).shape == (0, h * group, hd)
    assert hip.paged_append(k, v, table, empty[:, :h], empty[:, :h], i32(starts), cu=cu, max_new=7) is None


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("hd,sink,window", [(64, 0, 0), (128, 0, 0), (256, 2, 40), (128, 5, 70)])
def test_what_is_not_attended_to_leaves_no_trace(hd, sink, window, new, bad):
    """Rows behind every token's own, between the sinks and the window, and of other pages hold numbers that are not finite, and so does one
    row of V that the later tokens attend to: it makes the outputs of its columns what it is, of these tokens alone."""
    from diffcache_amd import _hip as hip
    h, group, page, n = 1, 3, 32, 333 + new
    k, v, table, g = build(1, h, hd, page, [n], 3)
    start = n - new
    at = lambda r: (int(table[0, r // page]), 0, r % page)  # noqa: E731
    if window:
        for r in range(sink, start - window + 1):
            k[at(r)], v[at(r)] = bad, bad
    mine = None
    if new > 1:
        mine = start + new // 2                # that token and the later ones attend to this row
        v[at(mine)][hd // 4:hd // 2] = bad
    q = tokens_of(1, new, h, group, hd, g)
    out, lse = hip.paged_attn(q, k, v, table, i32([start]), n_sink=sink, window=window, want_lse=True)
    clean = v.clone()
    if mine is not None:
        clean[at(mine)][hd // 4:hd // 2] = 0
    want = ref.attend(q[0], k, clean, table, [(0, new, start)], table.shape[1] * page, hd ** -0.5, sink, window)
    got = out[0].clone()
    if mine is not None:
        touched = got[new // 2:, :, hd // 4:hd // 2]
        assert (touched.isnan() if bad != bad else touched == bad).all()
        got[new // 2:, :, hd // 4:hd // 2] = want[0][new // 2:, :, hd // 4:hd // 2].to(torch.bfloat16)
    check(got, lse[0], want, 2.0 ** -8, hd)


@pytest.mark.parametrize("new", NEW)
def test_numbers_that_are_not_finite_where_they_are_attended_to(new):
    from diffcache_amd import _hip as hip
    h, group, hd, page, n = 2, 2, 128, 16, 600
    k, v, table, g = build(1, h, hd, page, [n + new], 4)
    at = lambda head, r: (int(table[0, r // page]), head, r % page)  # noqa: E731
    q = tokens_of(1, new, h, group, hd, g)
    k[at(0, 77)][5] = math.nan                 # head 0: everything
    v[at(1, 200)][3], v[at(1, 201)][4], v[at(1, 300)][9] = math.inf, -math.inf, math.nan
    v[at(1, 10)][50], v[at(1, 500)][50] = math.inf, -math.inf
    out, lse = hip.paged_attn(q, k, v, table, i32([n]), want_lse=True)
    assert out[..., :group, :].isnan().all() and lse[..., :group].isnan().all()
    rest = out[..., group:, :]
    assert (rest[..., 3] == math.inf).all() and (rest[..., 4] == -math.inf).all() and rest[..., 9].isnan().all() and rest[..., 50].isnan().all()
    keep = [c for c in range(hd) if c not in (3, 4, 9, 50)]
    assert rest[..., keep].isfinite().all() and lse[..., group:].isfinite().all()
    # logits beyond fp32: -inf weighs nothing, +inf makes its head NaN
    k.nan_to_num_(0), v.nan_to_num_(0)
    q.fill_(1e30)
    k[at(0, 3)] = -1e30
    k[at(1, 3)] = 1e30
    out, lse = hip.paged_attn(q, k, v, table, i32([n]), scale=1.0, want_lse=True)
    assert out[..., group:, :].isnan().all() and not out[..., :group, :].isnan().any()


@pytest.mark.parametrize("new", NEW)
def test_logits_of_minus_infinity_alone(new):
    from diffcache_amd import _hip as hip
    k, v, table, g = build(1, 1, 64, 16, [40 + new], 5)
    k.fill_(-1e30), v.fill_(1)
    q = torch.full((1, new, 2, 64), 1e30, dtype=torch.bfloat16, device=DEV)
    out, lse = hip.paged_attn(q, k, v, table, i32([40]), want_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_peaked_and_growing_logits(hd, new):
    """Logits of some hundreds, growing along the rows, so that the maximum moves again and again, and one row that outweighs all."""
    from diffcache_amd import _hip as hip
    h, group, page, n = 1, 4, 64, 1500
    k, v, table, g = build(1, h, hd, page, [n + new], 6)
    q = tokens_of(1, new, h, group, hd, g)
    direction = bf((hd,), g)
    r = torch.arange(n + new, device=DEV)
    k[table[0].long()[r // page], 0, r % page] = (direction * (r[:, None].float() / n * 6 - 3)).to(torch.bfloat16)
    q[:] = direction * 2
    q[..., 1, :] *= -1
    out, lse = hip.paged_attn(q, k, v, table, i32([n]), want_lse=True)
    want = ref.attend(q[0], k, v, table, [(0, new, n)], table.shape[1] * page, hd ** -0.5)
    # |q k| scale = 2 * 3 * sqrt(hd) = 96 at most here: hd products in fp32 off by hd 2^-24 of that, 256 * 96 * 2^-24 = 1.5e-3
    live = (out[0].double() - want[0]).abs()
    assert (live <= 2.0 ** -8 * want[0].abs() + (2.0 ** -8 + 3e-3) * want[2]).all()
    assert ((lse[0].double() - want[1]).abs() <= 3e-3).all()


def test_pools_of_more_than_32_bits():
    """Pages whose numbers lie past 2^32 bytes and past 2^31 numbers."""
    from diffcache_amd import _hip as hip
    h, hd, page, group = 2, 128, 64, 2
    n_pages = (1 << 31) // (h * page * hd) + 40
    k, v = (torch.empty((n_pages, h, page, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    table = i32([[n_pages - 1, 3, n_pages - 30, n_pages // 2 + 1]])
    g = torch.Generator(device=DEV).manual_seed(8)
    seq = 4 * page
    x = bf((1, seq, h, hd), g), bf((1, seq, h, hd), g)
    hip.paged_append(k, v, table, *x)
    for src, pool in zip(x, (k, v)):
        assert torch.equal(pool[table[0].long()].transpose(0, 1).flatten(1, 2), src[0].transpose(0, 1))
    for new in NEW:
        q = tokens_of(1, new, h, group, hd, g)
        out, lse = hip.paged_attn(q, k, v, table, i32([seq - new]), want_lse=True)
        small_k, small_v = (p[table[0].long()].clone() for p in (k, v))
        again = hip.paged_attn(q, small_k, small_v, i32([[0, 1, 2, 3]]), i32([seq - new]), want_lse=True)
        assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("new", NEW)
@pytest.mark.parametrize("layout", ["heads first", "k and v together", "wide pages"])
def test_other_layouts_of_pages(layout, new):
    from diffcache_amd import _hip as hip
    h, hd, page, group, n = 3, 64, 16, 2, 150
    k, v, table, g = build(2, h, hd, page, [n, 90 + new], 9)
    k.nan_to_num_(1), v.nan_to_num_(1)
    if layout == "heads first":
        a, b = (torch.empty((h, k.shape[0], page, hd), dtype=torch.bfloat16, device=DEV).transpose(0, 1) for _ in range(2))
    elif layout == "k and v together":
        both = torch.empty((k.shape[0], 2, h, page, hd), dtype=torch.bfloat16, device=DEV)
        a, b = both[:, 0], both[:, 1]
    else:
        a, b = (torch.empty((k.shape[0], h + 2, page * 2, hd), dtype=torch.bfloat16, device=DEV)[:, 1:h + 1, page:] for _ in range(2))
    a.copy_(k), b.copy_(v)
    wide = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    q = tokens_of(2, new, h, group, hd, g)
    src = bf((2, h * group + 2, new, hd), g)   # heads before tokens, and more of them
    src[:, 1:1 + h * group] = q.transpose(1, 2)
    odd = src[:, 1:1 + h * group].transpose(1, 2)
    starts = i32([n - new, 90])
    want = hip.paged_attn(q, k, v, table, starts, want_lse=True)
    got = hip.paged_attn(odd, a, b, wide[:, :table.shape[1]], starts, want_lse=True)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])
    nk, nv = bf((2, new, h, hd), g), bf((2, new, h, hd), g)
    inv = torch.rand((hd // 2,), generator=g, device=DEV)
    one = hip.paged_append(k, v, table, nk, nv, starts, q=q, inv_freq=inv)
    two = hip.paged_append(a, b, wide[:, :table.shape[1]], nk.transpose(1, 2).contiguous().transpose(1, 2), nv, starts, q=odd, inv_freq=inv)
    assert torch.equal(one, two) and torch.equal(a, k) and torch.equal(b, v)
    # what no alignment allows is copied
    shifted = torch.empty((q.numel() + 3,), dtype=torch.bfloat16, device=DEV)[3:].view(q.shape)
    shifted.copy_(q)
    assert torch.equal(hip.paged_append(a, b, table, nk, nv, starts, q=shifted, inv_freq=inv), one)


def test_queries_rotated_in_place():
    from diffcache_amd import _hip as hip
    k, v, table, g = build(2, 2, 128, 16, [40, 40], 10)
    nk, nv, q = bf((2, 30, 2, 128), g), bf((2, 30, 2, 128), g), bf((2, 30, 6, 128), g)
    inv = torch.rand((64,), generator=g, device=DEV)
    want = hip.paged_append(k, v, table, nk, nv, i32([3, 9]), q=q, inv_freq=inv)
    assert hip.paged_append(k, v, table, nk, nv, i32([3, 9]), q=q, q_out=q, inv_freq=inv) is q
    assert torch.equal(q, want)


def test_rows_without_a_page_are_not_written():
    from diffcache_amd import _hip as hip
    k, v, table, g = build(3, 2, 64, 16, [64, 64, 64], 11)
    before = k.clone(), v.clone()
    table[0, 1], table[1, 1], table[2, 1] = -1, k.shape[0], -2 ** 31
    nk, nv, q = bf((3, 40, 2, 64), g), bf((3, 40, 2, 64), g), bf((3, 40, 2, 64), g)
    inv = torch.rand((32,), generator=g, device=DEV)
    # rows 12 .. 51: those of the second page (16 .. 31) have none; sequence 2 begins behind the table's last row but eight
    out = hip.paged_append(k, v, table, nk, nv, i32([12, 12, 56]), q=q, inv_freq=inv)
    for i, start in enumerate([12, 12, 56]):
        for t in range(40):
            where = ref.place(table[i].tolist(), start + t, 16, k.shape[0])
            if where is not None:
                assert torch.equal(v[where[0], :, where[1]], nv[i, t])
                before[1][where[0], :, where[1]] = nv[i, t]
                before[0][where[0], :, where[1]] = k[where[0], :, where[1]]
        pos = torch.arange(start, start + 40, device=DEV)[:, None]
        assert ((out[i].double() - ref.rotate(q[i], pos, inv)).abs() <= 2.0 ** -8 * 4).all()       # queries are rotated all the same
    assert torch.equal(v.nan_to_num(7), before[1].nan_to_num(7)) and torch.equal(k.nan_to_num(7), before[0].nan_to_num(7))


@pytest.mark.parametrize("far", [1 << 20, (1 << 30) - 100, -(1 << 31)])
def test_angles_of_far_positions(far):
    from diffcache_amd import _hip as hip
    k, v, table, g = build(1, 1, 64, 16, [16], 12)
    x = bf((1, 16, 1, 64), g)
    inv = (1e4 ** (-torch.arange(32, device=DEV) / 32)).float()
    pos = (far + torch.arange(16, device=DEV)).to(torch.int32)[None]
    out = hip.paged_append(k, v, table, x, x, q=x, inv_freq=inv, pos=pos)
    want = ref.rotate(x[0], pos[0, :, None], inv)
    # the pairs' magnitude times the sine's error, and the product's in 64 bits: 2^30 turns of 2^-52 each
    assert ((out[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * x.abs().max()).all()


def test_the_same_call_gives_the_same_bits():
    from diffcache_amd import _hip as hip
    k, v, table, g = build(3, 2, 128, 64, [3000, 17, 900], 13)
    for new in NEW:
        q = tokens_of(3, new, 2, 4, 128, g)
        starts = i32([3000 - new, max(17 - new, 0), 900 - new])
        first = hip.paged_attn(q, k, v, table, starts, want_lse=True)
        for _ in range(5):
            again = hip.paged_attn(q, k, v, table, starts, want_lse=True)
            assert all(torch.equal(a.nan_to_num(9), b.nan_to_num(9)) for a, b in zip(first, again))


def test_a_workspace_that_holds_anything_and_is_shared_in_turn():
    from diffcache_amd import _hip as hip
    k, v, table, g = build(2, 2, 128, 64, [4000, 1200], 14)
    for new in NEW:
        q = tokens_of(2, new, 2, 4, 128, g)
        starts = i32([4000 - new, 1200 - new])
        want = hip.paged_attn(q, k, v, table, starts)
        need = hip.paged_attn_workspace_bytes(2, 2, 4, 128, 4032, new)
        assert need > 0
        ws = torch.full((need + 4096,), 255, dtype=torch.uint8, device=DEV)
        assert torch.equal(hip.paged_attn(q, k, v, table, starts, workspace=ws[:need]), want)
        assert (ws[need:] == 255).all()
        assert torch.equal(hip.paged_attn(q, k, v, table, starts, workspace=ws), want)
        with pytest.raises(hip.DiffCacheError, match="needed"):
            hip.paged_attn(q, k, v, table, starts, workspace=ws[:need - 256])


def test_streams_and_replayed_graphs():
    """Append and attention on a stream of their own, and captured: replays go by what start, table, counts and the tensors hold then."""
    from diffcache_amd import _hip as hip
    b, h, group, hd, page = 3, 2, 4, 128, 32
    k, v, table, g = build(b, h, hd, page, [2000, 700, 64], 15)
    k.nan_to_num_(0), v.nan_to_num_(0)
    for new in NEW:
        x = [bf((b, new, n, hd), g) for n in (h, h, h * group)]
        inv = torch.rand((hd // 2,), generator=g, device=DEV)
        start, counts = i32([100, 30, 2]), i32([new, 1, 0])
        out, lse = torch.zeros((b, new, h * group, hd), dtype=torch.bfloat16, device=DEV), torch.zeros((b, new, h * group), device=DEV)
        turned = torch.zeros_like(out)

        def step():
            hip.paged_append(k, v, table, x[0], x[1], start, counts=counts, q=x[2], q_out=turned, inv_freq=inv)
            hip.paged_attn(turned, k, v, table, start, counts=counts, n_rows=2000, out=out, lse=lse)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        for turn in range(6):
            start.copy_(i32([100 + 300 * turn, 30 + 100 * turn, 2 + 3 * turn])), counts.copy_(i32([new, 1, new] if turn % 2 else [0, new, 1]))
            for t in x:
                t.copy_(bf(t.shape, g))
            table.copy_(table.flip(0) if turn == 3 else table)      # (sequences trade their pages; all of them have rows enough there or none)
            out.fill_(1), lse.fill_(2)
            graph.replay()
            if turn % 2:
                torch.cuda.synchronize()
            got = out.clone(), lse.clone(), turned.clone()
            out.fill_(1), lse.fill_(2)
            step()
            assert torch.equal(out, got[0]) and torch.equal(lse, got[1]) and torch.equal(turned, got[2])


def test_two_streams_at_once():
    from diffcache_amd import _hip as hip
    sets = [build(2, 2, 128, 64, [6000, 900], s) for s in (16, 17)]
    q = [bf((2, 8, 128), s[3]) for s in sets]
    start = i32([5999, 899])
    want = [hip.paged_attn(a, s[0], s[1], s[2], start) for a, s in zip(q, sets)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(hip.paged_attn(q[i], sets[i][0], sets[i][1], sets[i][2], start))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("n_b", [1, 2, 63, 64, 65, 200, 700])
def test_packed_tokens_of_many_sequences(n_b):
    """Every sequence's tiles are found: lengths of none, one and several tiles, more sequences than lanes, a beginning that is not the first token."""
    from diffcache_amd import _hip as hip
    h, group, hd, page = 1, 4, 64, 16
    gen = torch.Generator().manual_seed(n_b)
    counts = [int(x) for x in (torch.rand((n_b,), generator=gen) ** 4 * 70)]
    counts[n_b // 2] = 69
    k, v, table, g = build(n_b, h, hd, page, [c + 1 for c in counts], n_b)
    ends = [33]
    for c in counts:
        ends.append(ends[-1] + c)
    q = bf((ends[-1] + 7, h * group, hd), g)
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)
    hip.paged_attn(q, k, v, table, i32([1] * n_b), cu=i32(ends), max_new=70, out=out, lse=lse)
    want = ref.attend(q, k, v, table, ref.spans(n_b, [1] * n_b, ends, None, 70, q.shape[0]), table.shape[1] * page, hd ** -0.5)
    check(out, lse, want, 2.0 ** -8, hd)
    # fewer than a sequence has: the first of its tokens
    if n_b > 1:
        out.fill_(4)
        hip.paged_attn(q, k, v, table, i32([1] * n_b), cu=i32(ends), max_new=33, out=out, lse=lse)
        span = ref.spans(n_b, [1] * n_b, ends, None, 33, q.shape[0])
        want = ref.attend(q, k, v, table, span, table.shape[1] * page, hd ** -0.5)
        check(out, lse, want, 2.0 ** -8, hd)
        assert (out[want[0].isnan().any(-1).any(-1)] == 4).all()
