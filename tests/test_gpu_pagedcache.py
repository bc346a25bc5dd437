"""PagedCache: a model's layers over prompts, chunks, decode steps and captured steps, against 64 bits."""
import copy
import math

import pytest
import torch

from oracle import paged as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(layers=2, b=2, n=400, hkv=2, hq=8, hd=128, **more):
    from diffcache_amd import PagedCache
    return PagedCache(layers, b, n, hkv, hq, hd, **more)


def bf(shape, g):
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


class Rows:
    """What a cache holds of one layer: rotated bf16 keys (rounded as they are held) and values of every sequence."""

    def __init__(self, b, inv):
        self.k, self.v, self.inv = [None] * b, [None] * b, inv

    def rotate(self, x, start):
        if self.inv is None:
            return x.double()
        pos = torch.arange(start, start + x.shape[0], device=DEV)[:, None]
        return ref.rotate(x, pos, self.inv).to(torch.bfloat16).double()

    def add(self, i, k, v):
        start = 0 if self.k[i] is None else self.k[i].shape[0]
        k = self.rotate(k, start)
        self.k[i] = k if self.k[i] is None else torch.cat([self.k[i], k])
        self.v[i] = v.double() if self.v[i] is None else torch.cat([self.v[i], v.double()])
        return start

    def attend(self, i, q, p, group, sink=0, window=0):
        """q (hq, hd), already rotated, of the token at row p."""
        keep = [r for r in range(p + 1) if window == 0 or r > p - window or r < sink]
        got = [ref.attention(q[j * group:(j + 1) * group], self.k[i][keep, j], self.v[i][keep, j], 1 / math.sqrt(q.shape[-1]))
               for j in range(self.k[i].shape[1])]
        return torch.cat([x[0] for x in got]), torch.cat([x[2] for x in got])


def near(got, want, weight, rotated, bits):
    # the output's rounding and the weights'; keys and queries that the oracle rounds to another neighbour than the kernel (one in some
    # hundreds, by 2^-8 of a product each, 128 products of random sign) move a logit by 2^-8 |q k| sqrt(2 / 300) or so
    bound = 2.0 ** -8 * want.abs() + (bits + 2.0 ** -11.5 + (2.0 ** -7 if rotated else 0)) * weight
    err = (got.double() - want).abs()
    assert (err <= bound).all(), (err / bound).max()
    assert err.square().sum().sqrt() <= 4e-3 * want.square().sum().sqrt()


@pytest.mark.parametrize("rotated", [False, True])
@pytest.mark.parametrize("hd,page,sink,window", [(128, 16, 0, 0), (64, 64, 0, 0), (256, 32, 3, 70)])
@pytest.mark.parametrize("lens", [None, [150, 3]])
def test_prompts_chunks_and_steps(hd, page, sink, window, lens, rotated):
    layers, b, hkv, g, seq = 2, 2, 2, 4, 150
    inv = (1e4 ** (-torch.arange(hd // 2, device=DEV) / (hd // 2))).float() if rotated else None
    cache = make(layers, b, 400, hkv, hkv * g, hd, page_size=page, sink_len=sink, window=window, inv_freq=inv)
    assert cache.rotates == rotated
    gen = torch.Generator(device=DEV).manual_seed(9)
    rows = [Rows(b, inv) for _ in range(layers)]
    held = list(lens or [seq] * b)
    for layer in range(layers):
        k, v = bf((b, seq, hkv, hd), gen), bf((b, seq, hkv, hd), gen)
        assert cache.prefill_update_kv_cache(k, v, layer, lens=lens)[0] is k
        for i in range(b):
            rows[layer].add(i, k[i, :held[i]], v[i, :held[i]])
    assert cache.seq_len(0) == seq and cache.lens.tolist() == held

    def turned(layer, q, start):
        return rows[layer].rotate(q, start)

    for counts in ([20, 20], [1, 37], [0, 3]):          # chunks, padded to the longest
        t = max(counts)
        for layer in range(layers):
            q, k, v = bf((b, t, hkv * g, hd), gen), bf((b, t, hkv, hd), gen), bf((b, t, hkv, hd), gen)
            out = torch.full_like(q, 5.0)
            got = cache.extend_attention(layer, q, k, v, lens=None if counts[0] == t else counts, out=out)
            assert got is out
            for i in range(b):
                start = rows[layer].add(i, k[i, :counts[i]], v[i, :counts[i]]) if counts[i] else held[i]
                assert (out[i, counts[i]:] == 5).all()
                qr = turned(layer, q[i, :counts[i]], start) if counts[i] else None
                for n in range(counts[i]):
                    near(out[i, n], *rows[layer].attend(i, qr[n], start + n, g, sink, window), rotated, 2.0 ** -8)
        held = [x + c for x, c in zip(held, counts)]
        assert cache.lens.tolist() == held
    for step in range(3):
        for layer in range(layers):
            q, k, v = bf((b, 1, hkv * g * hd), gen), bf((b, 1, hkv, hd), gen), bf((b, 1, hkv, hd), gen)
            out = cache.decode_attention(layer, q, k, v)
            for i in range(b):
                start = rows[layer].add(i, k[i], v[i])
                qr = turned(layer, q[i].view(1, hkv * g, hd), start)[0]
                near(out[i], *rows[layer].attend(i, qr, start, g, sink, window), rotated, 2.0 ** -15)
        held = [x + 1 for x in held]
        assert cache.lens.tolist() == held
    assert cache.seq_len(0) == cache.seq_len_gpu(1) == max(held)
    k, v = cache.get_kvcache(1)
    for i in range(b):
        want = rows[1].k[i].transpose(0, 1)
        assert ((k[i, :, :held[i]].double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -16).all()
        assert torch.equal(v[i, :, :held[i]].double(), rows[1].v[i].transpose(0, 1))


def test_a_captured_step_is_right_on_every_replay():
    layers, b, hkv, g, hd, seq = 3, 2, 2, 4, 128, 90
    inv = (1e4 ** (-torch.arange(hd // 2, device=DEV) / (hd // 2))).float()
    captured, eager = (make(layers, b, 130, hkv, hkv * g, hd, page_size=16, inv_freq=inv) for _ in range(2))
    gen = torch.Generator(device=DEV).manual_seed(1)
    for layer in range(layers):
        k, v = bf((b, seq, hkv, hd), gen), bf((b, seq, hkv, hd), gen)
        for c in (captured, eager):
            c.prefill_update_kv_cache(k, v, layer, lens=[seq, 17])
    q = torch.zeros((b, hkv * g, hd), dtype=torch.bfloat16, device=DEV)
    nk, nv = (torch.zeros((b, 1, hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    outs = [torch.empty_like(q) for _ in range(layers)]
    captured.reserve(130)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                       # a step of its own, taken back
        for layer in range(layers):
            captured.decode_attention(layer, q, nk, nv, out=outs[layer])
        captured.lens.sub_(1)
        captured.advance_host_step(-1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for layer in range(layers):
            captured.decode_attention(layer, q, nk, nv, out=outs[layer])
    for step in range(40):
        q.copy_(bf(q.shape, gen)), nk.copy_(bf(nk.shape, gen)), nv.copy_(bf(nv.shape, gen))
        graph.replay()
        captured.advance_host_step()
        for layer in range(layers):
            want = eager.decode_attention(layer, q, nk, nv)
            err = (outs[layer].double() - want.double()).abs()
            # the same rows, cut for 130 of them and for those that there are: the sums' order, and each output's rounding
            assert (err <= 2.0 ** -7 * want.double().abs() + 1e-5).all()
        if step % 7 == 0:
            torch.cuda.synchronize()
            assert captured.lens.tolist() == eager.lens.tolist() == [seq + step + 1, 18 + step]
    assert captured.seq_len(0) == eager.seq_len(0) == 130
    with pytest.raises(AssertionError, match="full"):
        eager.decode_attention(0, q, nk, nv)
    with pytest.raises(AssertionError, match="pages"):
        captured.advance_host_step(20)


def test_a_shared_beginning():
    """Three sequences, two of them behind the first one's pages, against a cache where each has its own."""
    layers, b, hkv, g, hd, seq, page = 2, 3, 2, 2, 64, 70, 16
    shared = make(layers, b, 128, hkv, hkv * g, hd, page_size=page, num_pages=14)
    alone = make(layers, b, 128, hkv, hkv * g, hd, page_size=page)
    gen = torch.Generator(device=DEV).manual_seed(2)
    for layer in range(layers):
        k, v = bf((1, seq, hkv, hd), gen).expand(b, -1, -1, -1), bf((1, seq, hkv, hd), gen).expand(b, -1, -1, -1)
        shared.prefill_update_kv_cache(k, v, layer, lens=[seq, 0, 0])
        alone.prefill_update_kv_cache(k, v, layer, lens=[seq, 64, 32])
    shared.share_prefix(1, 0, 64)
    shared.share_prefix(2, 0, 32)
    assert shared.lens.tolist() == [70, 64, 32] and len(shared._free) == 14 - 5
    for counts in ([5, 20, 1], [1, 1, 1]):
        for layer in range(layers):
            t = max(counts)
            q, k, v = bf((b, t, hkv * g, hd), gen), bf((b, t, hkv, hd), gen), bf((b, t, hkv, hd), gen)
            outs = [torch.zeros_like(q) for _ in range(2)]
            for c, o in zip((shared, alone), outs):
                c.extend_attention(layer, q, k, v, lens=counts, out=o)
            assert torch.equal(*outs)
    with pytest.raises(AssertionError, match="taken back"):
        shared.advance_host_step(-30)
    # the first one begins anew: the others keep what they hold
    before = [shared.get_kvcache(layer) for layer in range(layers)]
    for layer in range(layers):
        shared.prefill_update_kv_cache(bf((b, 33, hkv, hd), gen), bf((b, 33, hkv, hd), gen), layer, lens=[33, 0, 0])
    assert shared.lens.tolist() == [33, 0, 0]
    shared.free(0)
    shared.free(1)
    shared.free(2)
    assert sorted(shared._free) == list(range(14)) and (shared.table == -1).all()
    del before


def test_a_prompt_of_one_sequence_leaves_shared_pages_alone():
    layers, b, hkv, hd, page = 1, 2, 1, 64, 16
    cache = make(layers, b, 64, hkv, 2, hd, page_size=page)
    gen = torch.Generator(device=DEV).manual_seed(3)
    k, v = bf((b, 32, hkv, hd), gen), bf((b, 32, hkv, hd), gen)
    cache.prefill_update_kv_cache(k, v, 0, lens=[32, 0])
    cache.share_prefix(1, 0, 32)
    kept = list(cache._pages[1])
    cache.prefill_update_kv_cache(bf((b, 32, hkv, hd), gen), v, 0, lens=[32, 32])
    # (both begin anew here: neither has the other's pages)
    assert not set(cache._pages[0]) & set(cache._pages[1]) and kept != cache._pages[0]


def test_a_refused_prompt_leaves_shared_pages_where_they_were():
    from diffcache_amd import _hip as hip
    cache = make(1, 2, 64, 1, 2, 64, page_size=16)
    gen = torch.Generator(device=DEV).manual_seed(5)
    k, v = bf((2, 40, 1, 64), gen), bf((2, 40, 1, 64), gen)
    cache.prefill_update_kv_cache(k, v, 0, lens=[40, 0])
    cache.share_prefix(1, 0, 32)
    rows, table, free = cache.get_kvcache(0), cache.table.clone(), sorted(cache._free)
    for bad in (lambda: cache.prefill_update_kv_cache(k.float(), v.float(), 0), lambda: cache.prefill_update_kv_cache(k, v, 0, pos=torch.zeros((2, 40), device=DEV)),
                lambda: cache.prefill_update_kv_cache(k.cpu(), v.cpu(), 0)):
        with pytest.raises(hip.DiffCacheError):
            bad()
        assert torch.equal(cache.table, table) and sorted(cache._free) == free and cache.lens.tolist() == [40, 32] and cache._lens == [40, 32]
        assert all(torch.equal(a, b) for a, b in zip(cache.get_kvcache(0), rows))
    q = bf((2, 2, 64), gen)
    for bad in (lambda: cache.decode_attention(0, q.float(), k[:, :1], v[:, :1]), lambda: cache.decode_attention(0, q, k[:, :1].float(), v[:, :1])):
        with pytest.raises(hip.DiffCacheError):
            bad()
        assert cache.lens.tolist() == [40, 32] and cache._lens == [40, 32]


def test_a_copied_cache_has_memory_of_its_own():
    cache = make(1, 1, 64, 1, 2, 64, page_size=16)
    gen = torch.Generator(device=DEV).manual_seed(4)
    k, v = bf((1, 20, 1, 64), gen), bf((1, 20, 1, 64), gen)
    cache.prefill_update_kv_cache(k, v, 0)
    other = copy.deepcopy(cache)
    q, nk = bf((1, 2, 64), gen), bf((1, 1, 1, 64), gen)
    a = cache.decode_attention(0, q, nk, nk).clone()
    assert cache.lens.tolist() == [21] and other.lens.tolist() == [20] and other.seq_len(0) == 20
    assert torch.equal(other.decode_attention(0, q, nk, nk), a)


def test_the_harness_decodes_over_pages():
    from diffcache_amd import harness
    got = harness.run(2, 2, 512, 64, 3, 2, True, hidden=512, hq=8, hkv=2, hd=64, inter=1024, cache_kind="paged")
    assert got["finite"] and got["config"]["cache"] == "paged"
    eager = harness.run(2, 2, 512, 64, 3, 2, True, graphs=False, hidden=512, hq=8, hkv=2, hd=64, inter=1024, cache_kind="paged")
    assert eager["finite"]
