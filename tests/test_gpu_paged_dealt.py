"""A long sequence among short ones: every one's outputs, and into how many parts the long one's rows are cut."""
import pytest
import torch

from oracle import paged as ref
from test_gpu_paged_attn import bf, build, check, i32

pytestmark = pytest.mark.gpu


def parts_written(ws, tile_rows, hd, heads):
    """Parts to a head whose statistics stand in a workspace of 255s: a slot has tile_rows x hd fp32 sums, and behind all slots' sums
    tile_rows pairs of fp32 statistics, both aligned to 256 bytes."""
    up = lambda n: (n + 255) // 256 * 256  # noqa: E731
    slots = next(n for n in range(ws.numel()) if up(n * tile_rows * hd * 4) + up(n * tile_rows * 8) >= ws.numel())
    acc = up(slots * tile_rows * hd * 4)
    assert acc + up(slots * tile_rows * 8) == ws.numel()
    stats = ws[acc:acc + slots * tile_rows * 8].view(slots, -1)
    written = int((stats != 255).any(-1).sum())
    assert written % heads == 0
    return written // heads


@pytest.mark.parametrize("new,step,least", [(1, 32, 4), (40, 64, 7)])
def test_a_long_sequence_among_short_ones_gets_most_of_the_blocks(new, step, least):
    """One of 4000 rows and seven of 16 (or as many as they have tokens).  A block takes all steps of a short one; the long one's are cut into
    parts of `least` steps or fewer, to the nearest number: at least half as many parts as that divides."""
    from diffcache_amd import _hip as hip
    h, group, hd, page = 2, 4, 128, 16
    short = max(16, new)
    lengths = [short] * 3 + [4000] + [short] * 4
    k, v, table, g = build(8, h, hd, page, lengths, 7)
    q = bf((8, new, h * group, hd), g)
    starts = i32([n - new for n in lengths])
    ws = torch.full((hip.paged_attn_workspace_bytes(8, h, group, hd, 4000, new),), 255, dtype=torch.uint8, device=q.device)
    out, lse = hip.paged_attn(q, k, v, table, starts, n_rows=4000, want_lse=True, workspace=ws)
    want = ref.attend(q.flatten(0, 1), k, v, table, [(i * new, new, n - new) for i, n in enumerate(lengths)], 4000, hd ** -0.5)
    check(out.flatten(0, 1), lse.flatten(0, 1), want, 2.0 ** -15 if new * group <= 16 else 2.0 ** -8, hd)
    tiles = 1 if new * group <= 16 else -(-new * group // 128)
    assert parts_written(ws, new * group if tiles == 1 else 128, hd, h) >= tiles * (4000 // step // least // 2)
