"""The paged entries at the ends of what their arguments may be, on the host: what is refused before any kernel runs."""
import ctypes

import pytest
import torch

from diffcache_amd import _hip as hip
from test_paged_host import P, append_args, attn_args, refused


@pytest.mark.parametrize("scale", [2.36e38, 2.4e38, 2.999e38, 3.4e38])
def test_scales_that_are_infinite_in_powers_of_two_are_refused(scale):
    """The kernels take scale times log2(e): of an infinite one a logit of 0 would be NaN."""
    refused(hip.lib.dc_paged_attn_bf16(bytes(attn_args(scale=scale)), None), "scale")


@pytest.mark.parametrize("section", [5, 63, 1])
def test_one_section_holds_all_frequencies(section):
    """As several do: of fewer the rest would go by a position that the caller did not name for them."""
    refused(hip.lib.dc_paged_append_bf16(bytes(append_args(pos=P, section=(ctypes.c_int * 4)(section))), None), "hold %d" % section)


@pytest.mark.parametrize("section", [0, 5, 33])
def test_one_section_of_another_size_is_refused_by_the_wrapper(section, monkeypatch):
    monkeypatch.setattr(hip, "_mx_dev", lambda t, name: t.data_ptr())
    monkeypatch.setattr(hip, "_device", lambda: -1)
    monkeypatch.setattr(hip, "_stream", lambda: 0)
    pool, x = torch.zeros((4, 2, 16, 64), dtype=torch.bfloat16), torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(hip.DiffCacheError, match="hold"):
        hip.paged_append(pool, pool.clone(), torch.zeros((3, 5), dtype=torch.int32), x, x, inv_freq=torch.zeros(32), sections=(section,),
                         pos=torch.zeros((3, 1), dtype=torch.int32))
