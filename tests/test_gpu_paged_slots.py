"""PagedCache: sequences of a running batch that end, and others that begin in their places."""
import pytest
import torch

from test_gpu_pagedcache import DEV, Rows, bf, make, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("replayed", [False, True])
def test_sequences_end_and_begin_in_a_running_batch(replayed):
    """Eager steps, and one graph whose replays go by what was freed and filled since it was captured; the pool has no pages for a sequence
    that ended."""
    layers, b, hkv, g, hd, seq = 2, 3, 2, 4, 128, 90
    c = make(layers, b, 130, hkv, hkv * g, hd, page_size=16, num_pages=24)
    gen = torch.Generator(device=DEV).manual_seed(21)
    rows = [Rows(b, None) for _ in range(layers)]
    held = [seq, 50, 17]
    for layer in range(layers):
        k, v = bf((b, seq, hkv, hd), gen), bf((b, seq, hkv, hd), gen)
        c.prefill_update_kv_cache(k, v, layer, lens=held)
        for i in range(b):
            rows[layer].add(i, k[i, :held[i]], v[i, :held[i]])

    def free(i):
        c.free(i)
        held[i] = 0
        for r in rows:
            r.k[i] = r.v[i] = None

    q = [torch.zeros((b, hkv * g, hd), dtype=torch.bfloat16, device=DEV) for _ in range(layers)]
    nk, nv = ([torch.zeros((b, 1, hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(layers)] for _ in range(2))
    outs = [torch.zeros_like(x) for x in q]
    lses = [torch.zeros(x.shape[:2], device=DEV) for x in q]

    def step():
        for layer in range(layers):
            c.decode_attention(layer, q[layer], nk[layer], nv[layer], out=outs[layer], lse=lses[layer])

    free(1)
    c.reserve(130)                                     # 18 of the 24 pages: none of sequence 1
    if replayed:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                  # a step of its own, taken back
            step()
            c.lens.sub_(c.live)
            c.advance_host_step(-1)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()

    def steps(n, live):
        for turn in range(n):
            for layer in range(layers):
                for t in (q[layer], nk[layer], nv[layer]):
                    t.copy_(bf(t.shape, gen))
                outs[layer].fill_(5), lses[layer].fill_(7)
            if replayed:
                graph.replay()
                c.advance_host_step()
            else:
                step()
            if turn % 2:
                torch.cuda.synchronize()
            for layer in range(layers):
                for i in range(b):
                    if i not in live:
                        assert (outs[layer][i] == 5).all() and (lses[layer][i] == 7).all()
                        continue
                    p = rows[layer].add(i, nk[layer][i], nv[layer][i])
                    near(outs[layer][i], *rows[layer].attend(i, q[layer][i].double(), p, g), False, 2.0 ** -15)
            for i in live:
                held[i] += 1
            assert c.lens.tolist() == c._lens == held and c.live.tolist() == [int(i in live) for i in range(b)]

    steps(5, [0, 2])
    assert len(c._free) == 6 and (c.table[1] == -1).all()
    # a prompt joins in the place of the sequence that ended
    t = 37
    c.reserve([130, 60, 130])
    for layer in range(layers):
        x, k, v = bf((b, t, hkv * g, hd), gen), bf((b, t, hkv, hd), gen), bf((b, t, hkv, hd), gen)
        got = c.extend_attention(layer, x, k, v, lens=[0, t, 0])
        rows[layer].add(1, k[1], v[1])
        for n in range(t):
            near(got[1, n], *rows[layer].attend(1, x[1, n].double(), n, g), False, 2.0 ** -8)
    held[1] = t
    steps(4, [0, 1, 2])
    free(2)
    steps(3, [0, 1])
    free(0)
    free(1)
    steps(2, [])
    assert sorted(c._free) == list(range(24))


@pytest.mark.parametrize("rotated", [False, True])
def test_those_that_share_a_beginning_keep_it_when_the_first_one_ends(rotated):
    """Three sequences share pages; the one that wrote them is freed, and a new prompt takes its place and the pages that no one holds any
    more.  The others' rows stay to the bit, and their next tokens attend to them."""
    layers, b, hkv, g, hd, page, seq = 2, 3, 2, 2, 64, 16, 70
    inv = (1e4 ** (-torch.arange(hd // 2, device=DEV) / (hd // 2))).float() if rotated else None
    c = make(layers, b, 128, hkv, hkv * g, hd, page_size=page, num_pages=14, inv_freq=inv)
    gen = torch.Generator(device=DEV).manual_seed(22)
    rows = [Rows(b, inv) for _ in range(layers)]
    for layer in range(layers):
        k, v = bf((b, seq, hkv, hd), gen), bf((b, seq, hkv, hd), gen)
        c.prefill_update_kv_cache(k, v, layer, lens=[seq, 0, 0])
        for i, n in enumerate([seq, 64, 32]):
            rows[layer].add(i, k[0, :n], v[0, :n])
    c.share_prefix(1, 0, 64)
    c.share_prefix(2, 1, 32)
    shared = c._pages[0][:4]

    def extend(counts):
        t = max(counts)
        for layer in range(layers):
            q, k, v = bf((b, t, hkv * g, hd), gen), bf((b, t, hkv, hd), gen), bf((b, t, hkv, hd), gen)
            out = c.extend_attention(layer, q, k, v, lens=counts)
            for i, n in enumerate(counts):
                if n:
                    start = rows[layer].add(i, k[i, :n], v[i, :n])
                    turned = rows[layer].rotate(q[i, :n], start)
                    for x in range(n):
                        near(out[i, x], *rows[layer].attend(i, turned[x], start + x, g), rotated, 2.0 ** -8)

    extend([9, 2, 20])
    mine = c._pages[0][4:]
    kept = [[x.clone() for x in c.get_kvcache(layer)] for layer in range(layers)]
    lens = list(c._lens)
    assert lens == [79, 66, 52]
    c.free(0)
    for r in rows:
        r.k[0] = r.v[0] = None
    assert set(mine) <= set(c._free) and not set(shared) & set(c._free)
    extend([75, 0, 0])                         # five pages, the freed one among them
    assert set(mine) <= set(c._pages[0]) and not set(shared) & set(c._pages[0])
    for layer in range(layers):
        for now, old in zip(c.get_kvcache(layer), kept[layer]):
            for i in (1, 2):
                assert torch.equal(now[i, :, :lens[i]], old[i, :, :lens[i]])
    extend([1, 30, 3])
    for layer in range(layers):
        q, k, v = bf((b, hkv * g, hd), gen), bf((b, 1, hkv, hd), gen), bf((b, 1, hkv, hd), gen)
        out = c.decode_attention(layer, q, k, v)
        for i in range(b):
            p = rows[layer].add(i, k[i], v[i])
            near(out[i], *rows[layer].attend(i, rows[layer].rotate(q[i][None], p)[0], p, g), rotated, 2.0 ** -15)
    assert c.lens.tolist() == c._lens == [77, 97, 56]
    # the second one lets go as well: the third one alone holds what it began with
    c.free(1)
    assert set(shared[2:]) <= set(c._free) and not set(shared[:2]) & set(c._free)
    now = c.get_kvcache(0)
    assert all(torch.equal(a[2, :, :52], o[2, :, :52]) for a, o in zip(now, kept[0]))
