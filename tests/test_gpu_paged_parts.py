"""How attention over pages deals its steps out: sequences of very unequal lengths, more of them than lanes, packed tokens, no row twice and none left out."""
import pytest
import torch

from oracle import paged as ref
from test_gpu_paged_attn import DEV, bf, build, check, i32

pytestmark = pytest.mark.gpu


def lengths_of(b, most, seed):
    g = torch.Generator().manual_seed(seed)
    n = (most ** torch.rand((b,), generator=g)).int().tolist()
    n[b // 2] = most
    return [max(x, 1) for x in n]


@pytest.mark.parametrize("b,most,hd,h,group", [(1, 9000, 128, 1, 4), (3, 9000, 64, 2, 7), (8, 5000, 256, 2, 4), (64, 4000, 128, 2, 2), (65, 4000, 64, 1, 4), (130, 2500, 128, 3, 1),
                                               (300, 1800, 64, 1, 16), (800, 900, 128, 2, 1)])
def test_one_token_of_unequal_sequences(b, most, hd, h, group):
    from diffcache_amd import _hip as hip
    lengths = lengths_of(b, most, b)
    k, v, table, g = build(b, h, hd, 32, lengths, seed=b)
    q = bf((b, h * group, hd), g)
    out, lse = hip.paged_attn(q, k, v, table, i32([n - 1 for n in lengths]), want_lse=True)
    want = ref.attend(q, k, v, table, [(i, 1, n - 1) for i, n in enumerate(lengths)], table.shape[1] * 32, hd ** -0.5)
    check(out, lse, want, 2.0 ** -15, hd)


@pytest.mark.parametrize("b,most,new,hd,h,group", [(2, 3000, 40, 128, 1, 4), (5, 4000, 90, 64, 2, 7), (70, 1500, 30, 128, 1, 4), (3, 2500, 60, 256, 1, 4), (1, 6000, 33, 128, 2, 4)])
def test_packed_tokens_of_unequal_sequences(b, most, new, hd, h, group):
    from diffcache_amd import _hip as hip
    lengths = lengths_of(b, most, b + 1)
    g0 = torch.Generator().manual_seed(b)
    counts = [min(n, int(x)) for n, x in zip(lengths, torch.randint(0, new + 1, (b,), generator=g0))]
    counts[b // 2] = new
    k, v, table, g = build(b, h, hd, 16, lengths, seed=b)
    ends = [3]
    for c in counts:
        ends.append(ends[-1] + c)
    total = ends[-1] + 5
    q = bf((total, h * group, hd), g)
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 9.0, device=DEV)
    starts = [n - c for n, c in zip(lengths, counts)]
    hip.paged_attn(q, k, v, table, i32(starts), cu=i32(ends), max_new=new, out=out, lse=lse)
    span = ref.spans(b, starts, ends, None, new, total)
    want = ref.attend(q, k, v, table, span, table.shape[1] * 16, hd ** -0.5)
    check(out, lse, want, 2.0 ** -8, hd)
    # what is no sequence's stays
    assert (out[:3] == 3).all() and (out[-5:] == 3).all() and (lse[:3] == 9).all() and (lse[-5:] == 9).all()


def counted(b, h, hd, page, lengths, seed):
    """Values that count: column c of row r is 1 where r % hd == c, else 0.  With queries of zeros every row weighs the same, so the
    outputs are the numbers of a token's rows of each remainder over that of its rows, exactly, but for their own rounding."""
    k, v, table, g = build(b, h, hd, page, lengths, seed)
    v.zero_()
    for i, n in enumerate(lengths):
        r = torch.arange(n, device=DEV)
        v[table[i].long()[r // page], :, r % page] = torch.nn.functional.one_hot(r % hd, hd).to(torch.bfloat16)[:, None]
    return k.nan_to_num_(0), v, table, g


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("sink,window", [(0, 0), (5, 33), (70, 500), (0, 1), (300, 64)])
@pytest.mark.parametrize("new", [1, 2, 70])
def test_every_row_counts_once(hd, page, sink, window, new):
    from diffcache_amd import _hip as hip
    lengths = [new, 63 + new, 64 + new, 777 + new, 5003]
    b, h, group = len(lengths), 1, 3
    k, v, table, g = counted(b, h, hd, page, lengths, 1)
    q = torch.zeros((b, new, h * group, hd), dtype=torch.bfloat16, device=DEV)
    out, lse = hip.paged_attn(q, k, v, table, i32([n - new for n in lengths]), n_sink=sink, window=window, want_lse=True)
    for i, n in enumerate(lengths):
        for t in range(new):
            p = n - new + t
            r = torch.arange(p + 1, device=DEV)
            if window:
                r = r[(r > p - window) | (r < sink)]
            share = torch.bincount(r % hd, minlength=hd).double() / r.numel()
            # sums of ones up to 5003 are exact; a division, and for parts two products and a sum, in fp32
            got = out[i, t].double()
            assert ((got - share).abs() <= 2.0 ** -8 * share * (1 + 2.0 ** -12)).all()
            assert ((lse[i, t].double() - torch.tensor(r.numel(), dtype=torch.float64).log()).abs() <= 1e-5).all()


def test_a_long_and_many_short_sequences_take_little_more_than_their_rows():
    """One of 4000 rows among seven of 16 gets most of the blocks: its item alone would be one of its parts' time many times over.  (That no
    item is lost shows in the results; here only that two layouts of one call agree to rounding.)"""
    from diffcache_amd import _hip as hip
    lengths = [16] * 3 + [4000] + [16] * 4
    k, v, table, g = build(8, 2, 128, 16, lengths, 7)
    q = bf((8, 8, 128), g)
    a = hip.paged_attn(q, k, v, table, i32([n - 1 for n in lengths]))
    one = hip.paged_attn(q[3:4], k, v, table[3:4], i32([3999]))
    assert ((a[3].double() - one[0].double()).abs() <= 2.0 ** -7 * one[0].double().abs() + 1e-6).all()


@pytest.mark.parametrize("lengths,new,hd,h,group", [
    ([5589] * 11, 37, 128, 4, 1),                                                          # 44 tiles: 11 parts each where 12 are nearer, 484 items for 512 places
    ([1500, 1471, 1441, 1501, 1483] * 10, 20, 256, 6, 4),                                  # 300 tiles of a share and a half each: two parts, 600 items in two rounds
    ([6000, 9000, 7000, 8000, 8500], 120, 128, 2, 4),                                      # four tiles of each sequence, cut differently
    ([2100] * 66, 30, 256, 3, 4),                                                          # more sequences than lanes: the nearest number
    ([4099] * 7, 1, 128, 8, 4), ([4099, 3000, 100, 4000, 3500], 1, 128, 8, 4),              # of one token: fewer parts than the nearest number, and as many
    ([3600, 3000, 2500, 4000, 3500, 2800] * 3, 1, 128, 4, 4),                              # more than 16 sequences
    ([2900], 1100, 256, 8, 8),                                                             # 552 tiles for 512 places: 512 whole, 40 cut
    ([3000, 2900, 2950, 2800, 2990], 1000, 256, 4, 4),                                     # 640 of five sequences: the last one's all, and none of the others'
    ([3000, 2900, 2950, 2800, 2990], 900, 256, 4, 4),                                      # 580: some of the last one's
    ([700] * 8 + [5000], 240, 256, 8, 8),                                                  # 1080, one sequence's much longer: none cut
    ([2000] * 10, 160, 256, 8, 4),                                                         # 400: two rounds would be no shorter than one
])
def test_every_row_counts_once_however_tiles_are_cut(lengths, new, hd, h, group):
    from diffcache_amd import _hip as hip
    k, v, table, g = counted(len(lengths), h, hd, 64, lengths, 2)
    q = torch.zeros((len(lengths), new, h * group, hd), dtype=torch.bfloat16, device=DEV)
    out, lse = hip.paged_attn(q, k, v, table, i32([n - new for n in lengths]), want_lse=True)
    for i, n in enumerate(lengths):
        r = torch.arange(1, n + 1, device=DEV)[-new:, None]                                # rows of each token
        share = ((r - torch.arange(hd, device=DEV) + hd - 1).div(hd, rounding_mode="floor").double() / r)[:, None]
        # (the bounds as above, of counts that are exact in fp32)
        assert ((out[i].double() - share).abs() <= 2.0 ** -8 * share * (1 + 2.0 ** -12)).all()
        assert ((lse[i].double() - r.double().log()).abs() <= 1e-5).all()


@pytest.mark.parametrize("sink,window", [(0, 0), (64, 900), (0, 1500)])
@pytest.mark.parametrize("counts", [[700, 0, 1000, 999, 1, 1000], [1000, 1000, 130, 1000, 1000, 1]])
def test_packed_tokens_whose_last_tiles_are_cut(counts, sink, window):
    """More tiles than run at once: whole ones first, the rest in parts, across sequences with and without tokens."""
    from diffcache_amd import _hip as hip
    lengths, hd, h, group = [2600, 2500, 2700, 2650, 2400, 2550], 256, 4, 4
    k, v, table, g = counted(len(lengths), h, hd, 64, lengths, 3)
    ends = [2]
    for c in counts:
        ends.append(ends[-1] + c)
    total = ends[-1] + 3
    q = torch.zeros((total, h * group, hd), dtype=torch.bfloat16, device=DEV)
    out, lse = torch.full_like(q, 3.0), torch.full(q.shape[:2], 9.0, device=DEV)
    hip.paged_attn(q, k, v, table, i32([n - c for n, c in zip(lengths, counts)]), cu=i32(ends), max_new=1000, n_sink=sink, window=window, out=out, lse=lse)
    assert (out[:2] == 3).all() and (out[-3:] == 3).all() and (lse[:2] == 9).all() and (lse[-3:] == 9).all()
    below = lambda n: (n[:, None] - torch.arange(hd, device=DEV) + hd - 1).div(hd, rounding_mode="floor").clamp(min=0)  # noqa: E731 (rows 0 .. n - 1 of each remainder)
    for i, (n, c) in enumerate(zip(lengths, counts)):
        p = torch.arange(n - c, n, device=DEV)
        first = (p - window + 1).clamp(min=0) if window else torch.zeros_like(p)
        sinks = torch.minimum(first, torch.full_like(p, sink if window else 0))
        have = below(p + 1) - below(first) + below(sinks)
        rows = (p + 1 - first + sinks).double()
        share = (have.double() / rows[:, None])[:, None]
        got = out[ends[i]:ends[i + 1]].double()
        # (the bounds as above)
        assert ((got - share).abs() <= 2.0 ** -8 * share * (1 + 2.0 ** -12)).all()
        assert ((lse[ends[i]:ends[i + 1]].double() - rows.log()[:, None]).abs() <= 1e-5).all()
