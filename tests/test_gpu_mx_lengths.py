"""Lengths that no sequence has, and which of them leave a sequence's rows alone."""
import numpy as np
import pytest
import torch

from oracle import mx as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def hip():
    from diffcache_amd import _hip
    return _hip


def stores(rng, b, h, n, hd, bits=(4, 8)):
    out = []
    for x in bits:
        codes, scale = ref.encode(rng.standard_normal((b, h, n, hd)), x)
        out.append(hip().MxStore(torch.from_numpy(codes).to(DEV), torch.from_numpy(scale).to(DEV)))
    return out


@pytest.mark.parametrize("n", [90, 2500])
@pytest.mark.parametrize("captured", [False, True])
def test_a_step_with_idle_sequences(n, captured):
    """Lengths of n_rows and more: nothing is written and all rows are attended to.  Negative ones count as 0 for the attention,
    whose token then is row 0; mx_append writes neither."""
    rng = np.random.default_rng(n)
    lens = [n, 3, 2**31 - 1, n + 5, 0, n - 1, -1, -2**31]
    b, h, hd = len(lens), 2, 128
    ks, vs = stores(rng, b, h, n, hd)
    q = torch.from_numpy(rng.standard_normal((b, 4 * h, hd))).to(torch.bfloat16).to(DEV)
    nk, nv = (torch.from_numpy(rng.standard_normal((b, h, hd))).to(torch.bfloat16).to(DEV) for _ in range(2))
    at = torch.tensor(lens, dtype=torch.int32, device=DEV)
    before = [(s.codes.clone(), s.scale.clone()) for s in (ks, vs)]

    def rows_written(s, was):
        changed = (s.codes != was[0]).any(-1) | (s.scale != was[1]).any(-1)
        assert torch.equal(changed.any(1), changed.all(1))       # of both heads or of none
        return [changed[i, 0].nonzero().flatten().tolist() for i in range(b)]

    def run(call):
        if not captured:
            return call()
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=side):
            got = call()
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
        return got
    run(lambda: hip().mx_append(ks, vs, nk, nv, at))
    for s, was in zip((ks, vs), before):
        assert rows_written(s, was) == [[], [3], [], [], [0], [n - 1], [], []]
        s.codes.copy_(was[0])
        s.scale.copy_(was[1])
    out = run(lambda: hip().mx_attn(q, ks, vs, at, new_k=nk, new_v=nv))
    for s, was in zip((ks, vs), before):
        assert rows_written(s, was) == [[], [3], [], [], [0], [n - 1], [0], [0]]
    after = torch.tensor([n, 4, n, n, 1, n, 1, 1], dtype=torch.int32, device=DEV)
    assert torch.equal(out, hip().mx_attn(q, ks, vs, after))
    # without a token negative lengths are none
    out = run(lambda: hip().mx_attn(q, ks, vs, at))
    assert not out[[4, 6, 7]].any() and out[0].any()
    assert torch.equal(out[[0, 2, 3]], hip().mx_attn(q, ks, vs)[[0, 2, 3]])
