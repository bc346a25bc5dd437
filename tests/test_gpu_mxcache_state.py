"""MxCache as an object: copies of it, and what a refused call leaves."""
import copy
import io

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rnd(g, *shape):
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


def through_a_file(cache):
    f = io.BytesIO()
    torch.save(cache, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("again", [copy.deepcopy, through_a_file])
@pytest.mark.parametrize("bits", [(4, 4), (8, 4)])
def test_a_copy_of_a_cache_decodes_on_its_own(again, bits):
    """A copy of a cache in use continues as the original does, and neither sees the other's rows."""
    from diffcache_amd import MxCache
    g = torch.Generator(device=DEV).manual_seed(12)
    cache = MxCache(2, 2, 60, 2, 4, 64, key_bits=bits[0], value_bits=bits[1])
    for layer in range(2):
        cache.prefill_update_kv_cache(rnd(g, 2, 40, 2, 64), rnd(g, 2, 40, 2, 64), layer, lens=[40, 11])
    tokens = [[(rnd(g, 2, 4, 64), rnd(g, 2, 2, 64), rnd(g, 2, 2, 64)) for _ in range(2)] for _ in range(7)]

    def step(c, token):
        return [c.decode_attention(layer, *token[layer]).clone() for layer in range(2)]
    for token in tokens[:2]:
        step(cache, token)
    other = again(cache)
    for a, b in zip(cache.kstore + cache.vstore, other.kstore + other.vstore):
        assert a.codes.data_ptr() != b.codes.data_ptr() and a.scale.data_ptr() != b.scale.data_ptr()
    for token in tokens[2:5]:
        for x, y in zip(step(cache, token), step(other, token)):
            assert torch.equal(x, y)
    # the copy alone goes on: the original's rows stay, and the copy's are its own
    before = [(s.codes.clone(), s.scale.clone()) for s in cache.kstore + cache.vstore]
    step(other, tokens[5])
    for s, (codes, scale) in zip(cache.kstore + cache.vstore, before):
        assert torch.equal(s.codes, codes) and torch.equal(s.scale, scale)
    want = step(cache, tokens[5])
    rest = step(cache, tokens[6])
    del cache
    for x, y in zip(step(other, tokens[6]), rest):
        assert torch.equal(x, y)
    assert other.seq_len(0) == 47 and other.lens.tolist() == [47, 18] and len(want) == 2


def test_a_refused_prefill_leaves_the_cache_as_it_was():
    from diffcache_amd import MxCache
    g = torch.Generator(device=DEV).manual_seed(5)
    cache = MxCache(2, 2, 80, 2, 8, 128)
    k, v = rnd(g, 2, 50, 2, 128), rnd(g, 2, 50, 2, 128)

    def state():
        return cache.lens.tolist(), cache.seq_len(0), cache.seq_len_gpu(0)

    def refusals():
        for lens in (None, [33, 7]):
            for a, b, error in ((k.float(), v.float(), RuntimeError), (k, v.half(), RuntimeError), (k[:1], v[:1], RuntimeError),
                                (k[:, :, :1], v[:, :, :1], RuntimeError), (k, v[:, :49], RuntimeError), (k[..., :64], v[..., :64], RuntimeError),
                                (k.cpu(), v.cpu(), RuntimeError), (k, v.cpu(), RuntimeError), (k[0], v[0], RuntimeError)):
                with pytest.raises(error):
                    cache.prefill_update_kv_cache(a, b, 0, lens=lens if a.shape[1] == 50 else None)
                yield
            with pytest.raises(IndexError):
                cache.prefill_update_kv_cache(k, v, 2, lens=lens)
            yield
        for lens in ([50], [51, 3], [-1, 3], [1, 2, 3]):
            with pytest.raises(AssertionError, match="lens"):
                cache.prefill_update_kv_cache(k, v, 0, lens=lens)
            yield
    for _ in refusals():
        assert state() == ([0, 0], 0, 0)
    for layer in range(2):
        cache.prefill_update_kv_cache(k, v, layer, lens=[20, 9])
    other = copy.deepcopy(cache)
    for _ in refusals():
        assert state() == ([20, 9], 20, 20)
    for layer in range(2):
        token = rnd(g, 2, 8, 128), rnd(g, 2, 2, 128), rnd(g, 2, 2, 128)
        assert torch.equal(cache.decode_attention(layer, *token), other.decode_attention(layer, *token))
    assert state() == ([21, 10], 21, 21) and cache.get_kvcache(0)[0].shape == (2, 2, 21, 128)
