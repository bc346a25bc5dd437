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
