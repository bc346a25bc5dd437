"""The paged entries at the ends of what their arguments may be, on the host: what is refused before any kernel runs."""
import pytest

from diffcache_amd import _hip as hip
from test_paged_host import attn_args, refused


@pytest.mark.parametrize("scale", [2.36e38, 2.4e38, 2.999e38, 3.4e38])
def test_scales_that_are_infinite_in_powers_of_two_are_refused(scale):
    """The kernels take scale times log2(e): of an infinite one a logit of 0 would be NaN."""
    refused(hip.lib.dc_paged_attn_bf16(bytes(attn_args(scale=scale)), None), "scale")
