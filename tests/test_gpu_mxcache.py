"""MxCache: a model's layers over prompts, decode steps and captured steps, against 64 bits."""
import math

import numpy as np
import pytest
import torch

from oracle import mx as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(layers=2, b=2, n=400, hkv=2, hq=8, hd=128, **more):
    from diffcache_amd import MxCache
    return MxCache(layers, b, n, hkv, hq, hd, **more)


def prompt(b, seq, h, hd, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn((b, seq, h, hd), generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]


def want(q, rows_k, rows_v, bits_k, bits_v, sink=0, window=0):
    """One unit: q (g, hd) over bf16 rows as the cache holds them."""
    k, v = (ref.decode(*ref.encode(x, bits)) for x, bits in ((rows_k, bits_k), (rows_v, bits_v)))
    keep = ref.attended(len(k), sink, window)
    out, lse, weight, _ = ref.attention(q, k[keep], v[keep], 1 / math.sqrt(q.shape[-1]))
    return out, weight


@pytest.mark.parametrize("bits,hd,sink,window", [((4, 4), 128, 0, 0), ((8, 4), 64, 0, 0), ((4, 8), 256, 2, 130)])
@pytest.mark.parametrize("lens", [None, [150, 3]])
def test_steps_of_all_layers(bits, hd, sink, window, lens):
    layers, b, hkv, g, seq = 2, 2, 2, 4, 150
    cache = make(layers, b, 400, hkv, hkv * g, hd, key_bits=bits[0], value_bits=bits[1], sink_len=sink, window=window)
    rows = []
    for layer in range(layers):
        k, v = prompt(b, seq, hkv, hd, layer)
        assert cache.prefill_update_kv_cache(k, v, layer, lens=lens)[0] is k
        rows.append([[x[i, :(lens or [seq] * b)[i]].double().cpu().numpy() for i in range(b)] for x in (k, v)])
    assert cache.seq_len(0) == seq and cache.lens.tolist() == (lens or [seq] * b)
    g_ = torch.Generator(device=DEV).manual_seed(9)
    for step in range(4):
        for layer in range(layers):
            q = torch.randn((b, 1, hkv * g * hd), generator=g_, device=DEV).to(torch.bfloat16)
            nk, nv = (torch.randn((b, 1, hkv, hd), generator=g_, device=DEV).to(torch.bfloat16) for _ in range(2))
            out = cache.decode_attention(layer, q, nk, nv)
            for x, new in zip(rows[layer], (nk, nv)):
                for i in range(b):
                    x[i] = np.concatenate([x[i], new[i].double().cpu().numpy()])
            qx = q.double().cpu().numpy().reshape(b, hkv, g, hd)
            for i in range(b):
                for h in range(hkv):
                    y, weight = want(qx[i, h], rows[layer][0][i][:, h], rows[layer][1][i][:, h], *bits, sink, window)
                    got = out[i].double().cpu().numpy().reshape(hkv, g, hd)[h]
                    # (output rounding; P, exp2 and fp32 sums of some 150 rows and logits of a few tens)
                    assert (np.abs(got - y) <= 2.0 ** -8 * np.abs(y) + 2.0 ** -13 * weight).all()
        assert cache.lens.tolist() == [(lens or [seq] * b)[i] + step + 1 for i in range(b)]
    assert cache.seq_len(0) == cache.seq_len_gpu(1) == seq + 4
    k, v = cache.get_kvcache(1)
    for i in range(b):
        n = len(rows[1][0][i])
        held = ref.decode(*ref.encode(rows[1][0][i].transpose(1, 0, 2), bits[0]))
        assert np.array_equal(k[i, :, :n].double().cpu().numpy(), held)


def test_a_captured_step_is_right_on_every_replay():
    layers, b, hkv, g, hd, seq = 3, 2, 2, 4, 128, 90
    caches = [make(layers, b, 130, hkv, hkv * g, hd) for _ in range(2)]
    for layer in range(layers):
        k, v = prompt(b, seq, hkv, hd, layer)
        for c in caches:
            c.prefill_update_kv_cache(k, v, layer, lens=[seq, 17])
    q = torch.zeros((b, hkv * g, hd), dtype=torch.bfloat16, device=DEV)
    nk, nv = (torch.zeros((b, 1, hkv, hd), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    outs = [torch.empty_like(q) for _ in range(layers)]
    captured, eager = caches
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for layer in range(layers):
            captured.decode_attention(layer, q, nk, nv, out=outs[layer])
    assert captured.lens.tolist() == [seq, 17] and captured.seq_len(0) == seq
    for step in range(40):
        for t in (q, nk, nv):
            t.copy_(torch.randn(t.shape, device=DEV))
        graph.replay()
        captured.advance_host_step()
        for layer in range(layers):
            out = eager.decode_attention(layer, q, nk, nv)
            # (the two cut the rows otherwise: equal up to the rounding of sums in another order)
            d = (out.double() - outs[layer].double()).abs()
            assert (d <= 2.0 ** -7 * out.double().abs() + 2.0 ** -12).all(), (step, layer)
        if step % 7 == 0:
            torch.cuda.synchronize()
        assert torch.equal(captured.lens, eager.lens)
    for x, y in zip(captured.kstore + captured.vstore, eager.kstore + eager.vstore):
        assert torch.equal(x.codes, y.codes) and torch.equal(x.scale, y.scale)
    assert captured.seq_len(0) == eager.seq_len(0) == 130
    # the first sequence is full: the next step has no row for it
    with pytest.raises(AssertionError, match="full"):
        eager.decode_attention(0, q, nk, nv)
    with pytest.raises(AssertionError, match="rows"):
        captured.advance_host_step()
    before = captured.kstore[0].codes.clone()
    graph.replay()                                   # one too many writes nothing there and attends to what there is
    assert torch.equal(captured.kstore[0].codes[0], before[0]) and not torch.isnan(outs[0].float()).any()
    assert not torch.equal(captured.kstore[0].codes[1, :, 57], before[1, :, 57])   # the shorter one has room
    eager.advance_host_step(-1)                      # a token taken back
    eager.lens.sub_(1)
    eager.decode_attention(0, q, nk, nv)


def test_refusals():
    cache = make()
    k, v = prompt(2, 50, 2, 128, 0)
    with pytest.raises(AssertionError, match="empty or longer"):
        cache.prefill_update_kv_cache(k[:, :0], v[:, :0], 0)
    with pytest.raises(AssertionError, match="empty or longer"):
        cache.prefill_update_kv_cache(*prompt(2, 401, 2, 128, 0), 0)
    for lens in ([50], [51, 3], [-1, 3]):
        with pytest.raises(AssertionError, match="lens"):
            cache.prefill_update_kv_cache(k, v, 0, lens=lens)
    for bad in (dict(layers=0), dict(n=0), dict(hq=7), dict(window=-1)):
        with pytest.raises(AssertionError):
            make(**bad)
    for bad in (dict(hd=96), dict(key_bits=5)):
        with pytest.raises(RuntimeError):
            make(**bad)
    with pytest.raises(RuntimeError, match="bf16"):
        cache.prefill_update_kv_cache(k.float(), v.float(), 0)
    cache.prefill_update_kv_cache(k, v, 0)
    with pytest.raises(RuntimeError, match="new_k"):
        cache.decode_attention(0, torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=DEV), k[:, :1, :1], v[:, :1])


def test_harness_decodes_over_it():
    """The synthetic decoder's step over an MxCache, eager and with captured halves: what every layer attends to against 64 bits
    over the rows that the cache holds."""
    from diffcache_amd import MxCache
    from diffcache_amd.harness import GraphedDecoder, SyntheticLlama, synthetic_prompt_cache
    layers, b, ctx, hidden, hq, hkv, hd, inter = 2, 2, 300, 256, 8, 2, 64, 512
    model = SyntheticLlama(layers, hidden, hq, hkv, hd, inter, device=DEV)
    calls = []

    class Checked(MxCache):
        def decode_attention(self, layer_idx, queries, key_states, value_states, out=None, lse=None):
            before = self.seq_len(layer_idx)
            got = super().decode_attention(layer_idx, queries, key_states, value_states, out=out, lse=lse)
            n = before + 1
            k, v = (x.double().cpu().numpy() for x in hip_rows(self, layer_idx, n))
            q = queries.double().cpu().numpy().reshape(b, hkv, hq // hkv, hd)
            y = got.double().cpu().numpy().reshape(b, hkv, hq // hkv, hd)
            for i in range(b):
                for h in range(hkv):
                    ref_out, _, weight, logit = ref.attention(q[i, h], k[i, h], v[i, h], hd ** -0.5)
                    rel = 2 * (hd + 4) * 2.0 ** -24 * logit + 2.0 ** -15 + 2 * n * 2.0 ** -24
                    assert (np.abs(y[i, h] - ref_out) <= 2.0 ** -8 * np.abs(ref_out) + weight * rel[:, None]).all()
            token = key_states.double().cpu().numpy().reshape(b, hkv, hd)
            assert np.array_equal(k[:, :, -1], ref.decode(*ref.encode(token, 8)))
            calls.append(layer_idx)
            return got

    def hip_rows(cache, layer, n):
        from diffcache_amd import _hip
        return _hip.mx_gather_rows(cache.kstore[layer], cache.vstore[layer], n_idx=n)

    cache = Checked(layers, b, ctx + 40, hkv, hq, hd, key_bits=8, value_bits=4)
    synthetic_prompt_cache(cache, ctx)
    x = torch.randn((b, hidden), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    y = model.decode_step(cache, x)
    assert calls == [0, 1] and cache.seq_len(0) == ctx + 1 and torch.isfinite(y.float()).all()
    dec = GraphedDecoder(model, cache, b)
    z = dec.decode_step(x)
    assert calls == [0, 1, 0, 1] and cache.lens.tolist() == [ctx + 2] * b and torch.isfinite(z.float()).all()
