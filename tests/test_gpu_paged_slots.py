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
