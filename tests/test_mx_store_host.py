"""Stores and caches of the block-scaled kind without a GPU: copies, and calls that are refused before anything is launched."""
import copy
import itertools
import pickle
import struct

import pytest
import torch

from diffcache_amd import _hip as hip


@pytest.fixture
def on_cpu(monkeypatch):
    """Stores of CPU tensors, for what the host does with them alone."""
    monkeypatch.setattr(hip, "_mx_dev", lambda t, name: t.data_ptr())
    monkeypatch.setattr(hip, "_device", lambda: -1)


def addresses(store):
    return struct.unpack_from("@2P", store.args)


@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda s: pickle.loads(pickle.dumps(s)), lambda s: copy.deepcopy([s])[0]])
def test_a_copied_store_names_its_own_memory(on_cpu, again):
    room = torch.arange(2 * 3 * 2 * 9 * 64, dtype=torch.int64).to(torch.uint8).view(2, 3, 2, 9, 64)
    store = hip.MxStore(room[:, 1, :, 2:7], torch.ones((2, 2, 5, 4), dtype=torch.uint8))
    other = again(store)
    assert type(other) is hip.MxStore and addresses(other) == (other.codes.data_ptr(), other.scale.data_ptr())
    assert (addresses(other) == addresses(store)) == (again is copy.copy)
    assert torch.equal(other.codes, store.codes) and torch.equal(other.scale, store.scale)
    assert (other.shape, other.units, other.hd, other.bits) == (store.shape, store.units, store.hd, store.bits)
    # strides, room and bits go along
    assert struct.unpack("@2P4q2i", other.args)[2:] == struct.unpack("@2P4q2i", store.args)[2:]


@pytest.mark.parametrize("hkv,hq,message", [(2, 34, "query heads"), (1, 32, "query heads"), (2, 7, "multiple"), (0, 4, "multiple"),
                                            (2, 0, "multiple"), (-1, 4, "multiple")])
def test_heads_that_no_step_could_attend_with_are_refused_at_once(hkv, hq, message):
    """Before any memory is taken: where there is no GPU, anything later fails otherwise."""
    from diffcache_amd import MxCache
    with pytest.raises(AssertionError, match=message):
        MxCache(1, 1, 64, hkv, hq, 128)


def test_the_largest_group_is_the_library_s():
    store = hip.MxStoreArgs(1 << 20, 1 << 21, 4096, 4096, 256, 256, 4, 64)
    p = 1 << 22
    args = hip.MxAttnArgs(p, None, None, p, None, p, store, store, p, 1 << 30, 2, 2, hip.MX_MAX_GROUP + 1, 128, 64, 0, 0, 0.1)
    assert hip.lib.dc_mx_attn_bf16(bytes(args), None) == -22 and f"not in [1,{hip.MX_MAX_GROUP}]" in hip.lib.dc_last_error().decode()


def refused(rc, message):
    assert rc == -22 and message in hip.lib.dc_last_error().decode(), (rc, hip.lib.dc_last_error())


def long_store(n_rows, hd, bits=4):
    """A store of one unit that no kernel is launched on."""
    return bytes(hip.MxStoreArgs(1 << 20, 1 << 21, 0, 0, 0, 0, bits, n_rows))


@pytest.mark.parametrize("hd,rows_per", [(64, 128), (128, 64), (256, 32)])
def test_prompts_near_the_end_of_32_bits_are_refused(hd, rows_per):
    """A thread's row numbers, those past the end too, are ints: of the last block all have to be."""
    last, p = 2**31 - 1, 1 << 22
    s = long_store(last, hd)
    for seq, dst in ((last, 0), (last - 1, 1), (last - rows_per + 2, 0)):   # (the sum of seq and rows_per - 1 passes 2^31)
        refused(hip.lib.dc_mx_ingest_bf16(s, s, p, p, None, 1, seq, 1, hd, dst, 0, 0, 0, 0, 0, 0, None), "grid too large")
    for n in (last, last - 1):
        refused(hip.lib.dc_mx_gather_rows_bf16(s, s, None, p, p, 1, 1, n, 0, hd, 0, 0, 0, 0, None), "grid too large")


def test_more_blocks_than_a_launch_takes_are_refused():
    """2^24 blocks of 256 threads: one more thread than a launch counts."""
    p, b, h, hd = 1 << 22, 1 << 12, 1 << 11, 64
    s = bytes(hip.MxStoreArgs(1 << 20, 1 << 30, h * 160 * 32, 160 * 32, h * 160 * 2, 160 * 2, 4, 160))
    refused(hip.lib.dc_mx_ingest_bf16(s, s, p, p, None, b, 129, h, hd, 0, 0, 0, 0, 0, 0, 0, None), "grid too large")
    refused(hip.lib.dc_mx_gather_rows_bf16(s, s, None, p, p, b, h, 65, 0, hd, 0, 0, 0, 0, None), "grid too large")


def every_call(k, v, b, h, hd=128):
    """The calls that write, each with stores that nothing else is wrong with."""
    p = 1 << 22
    yield lambda: hip.lib.dc_mx_ingest_bf16(k, v, p, p, None, b, 1, h, hd, 0, 0, 0, 0, 0, 0, 0, None)
    yield lambda: hip.lib.dc_mx_append_bf16(k, v, p, p, p, b, h, hd, None)
    args = hip.MxAttnArgs(p, p, p, p, None, p, hip.MxStoreArgs.from_buffer_copy(k), hip.MxStoreArgs.from_buffer_copy(v), None, 0, b, h, 1,
                          hd, 1, 0, 0, 0.1)
    yield lambda: hip.lib.dc_mx_attn_bf16(bytes(args), None)


def store(b, h, n, cb, ch, sb, sh, bits=4):
    return bytes(hip.MxStoreArgs(1 << 20, 1 << 21, cb, ch, sb, sh, bits, n))


# strides in rows (64 and 4 bytes): batch, head; of units of 10 rows
@pytest.mark.parametrize("b,h,code,scale", [
    (3, 2, (20, 9), (20, 10)), (3, 2, (20, 10), (20, 9)), (3, 2, (19, 10), (20, 10)), (3, 2, (20, 10), (19, 10)), (3, 2, (10, 10), (20, 10)),
    (3, 2, (1, 30), (20, 10)), (5, 1, (9, 0), (10, 0)), (1, 4, (0, 10), (0, 3)), (2, 2, (15, 10), (20, 10)), (2, 3, (25, 10), (30, 10)),
    (3, 3, (10, 20), (30, 10)), (3, 1, (0, 0), (10, 0)), (1, 3, (0, 10), (0, 0)), (4, 7, (30, 45), (70, 10)),
])
def test_units_that_overlap_are_not_written(b, h, code, scale):
    good = store(b, h, 10, h * 640, 640, h * 40, 40)
    bad = store(b, h, 10, 64 * code[0], 64 * code[1], 4 * scale[0], 4 * scale[1])
    for k, v in ((good, bad), (bad, good)):
        for call in every_call(k, v, b, h):
            refused(call(), "share their rows")


@pytest.mark.parametrize("b,h,code,scale", [
    (3, 2, (20, 10), (20, 10)), (3, 2, (10, 30), (10, 30)), (3, 2, (100, 10), (25, 12)), (1, 4, (0, 10), (0, 10)), (1, 4, (3, 10), (1, 10)),
    (5, 1, (10, 0), (10, 1)), (2, 2, (15, 30), (10, 20)), (2, 3, (10, 20), (30, 10)), (1, 1, (0, 0), (0, 0)),
])
def test_units_that_lie_apart_are(b, h, code, scale):
    """Apart also where the units of one sequence lie between another's: refused nowhere (without a GPU the launch fails)."""
    s = store(b, h, 10, 64 * code[0], 64 * code[1], 4 * scale[0], 4 * scale[1])
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up")
    for call in every_call(s, s, b, h):
        assert call() == -5


def test_overlap_against_every_pair_of_units():
    """The rule against a comparison of all pairs, over small strides."""
    if torch.cuda.is_available():
        pytest.skip("the addresses are made up")
    for b, h, n in ((2, 3, 2), (3, 2, 3), (4, 4, 1)):
        for cb, ch in itertools.product(range(0, 9), repeat=2):
            rows = [i * cb + j * ch for i in range(b) for j in range(h)]
            apart = all(abs(x - y) >= n for x, y in itertools.combinations(rows, 2))
            s = store(b, h, n, 64 * cb, 64 * ch, 4 * h * n, 4 * n)
            rc = hip.lib.dc_mx_append_bf16(s, s, 1 << 22, 1 << 22, 1 << 22, b, h, 128, None)
            assert rc == (-5 if apart else -22), (b, h, n, cb, ch)


class NotReached:
    def __getattr__(self, name):
        if name == "dc_mx_attn_workspace_bytes":
            return lambda *a: 0
        raise AssertionError(f"{name} was called")


@pytest.fixture
def no_library(on_cpu, monkeypatch):
    """What a wrapper refuses by itself: a call that gets further fails."""
    monkeypatch.setattr(hip, "lib", NotReached())
    monkeypatch.setattr(hip, "_mx_stream", lambda k, v: 0)


def cpu_store(b=1, h=2, n=2000, hd=128, bits=4):
    return hip.MxStore(torch.zeros((b, h, n, hd * bits // 8), dtype=torch.uint8), torch.zeros((b, h, n, hd // 32), dtype=torch.uint8))


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 24), torch.zeros(1 << 12, dtype=torch.uint8)[::2],
                                       torch.zeros((2, 64), dtype=torch.float32).t()])
def test_a_workspace_with_gaps_or_overlaps_is_refused(no_library, workspace):
    """Its elements say nothing about the memory behind it."""
    s = cpu_store()
    q = torch.zeros((1, 8, 128), dtype=torch.bfloat16)
    with pytest.raises(hip.DiffCacheError, match="workspace must be contiguous"):
        hip.mx_attn(q, s, s, workspace=workspace)
    with pytest.raises(AssertionError, match="dc_mx_attn_bf16"):    # a plain one goes on
        hip.mx_attn(q, s, s, workspace=torch.zeros(1 << 12, dtype=torch.uint8))


def test_numbers_that_no_c_type_holds_are_refused(no_library):
    s = cpu_store()
    q = torch.zeros((1, 8, 128), dtype=torch.bfloat16)
    for bad in (dict(window=1 << 31), dict(n_sink=1 << 40), dict(n_sink=1.5), dict(window=1 << 64)):
        with pytest.raises(hip.DiffCacheError, match="does not fit"):
            hip.mx_attn(q, s, s, **bad)
    out = torch.zeros((1, 1, 1, 128), dtype=torch.bfloat16).expand(1, 2, (1 << 32) + 3, 128)
    for bad in (dict(n_idx=1 << 31), dict(n_idx=(1 << 32) + 3), dict(row_offset=1 << 63, n_idx=3), dict(row_offset=1 << 64, n_idx=3)):
        with pytest.raises(hip.DiffCacheError, match="too large"):   # (ctypes would take the low bits)
            hip.mx_gather_rows(s, None, out_k=out, **bad)
    long = [torch.empty((1, 1, 1 << 31, row), dtype=torch.uint8, device="meta") for row in (64, 4)]
    with pytest.raises(hip.DiffCacheError, match="does not fit"):
        hip.MxStore(*long)


def test_rows_past_any_row_are_refused_where_their_number_would_wrap():
    s = long_store(64, 128)
    for off in (1 << 62, 2**63 - 1):
        refused(hip.lib.dc_mx_gather_rows_bf16(s, s, 1 << 22, 1 << 22, 1 << 22, 1, 1, 1, 1, 128, off, 128, 128, 128, None), "bad sizes")


def test_a_store_without_heads_is_refused(no_library):
    s = cpu_store(h=0)
    with pytest.raises(hip.DiffCacheError, match="q must be"):
        hip.mx_attn(torch.zeros((1, 0, 128), dtype=torch.bfloat16), s, s)


def test_a_store_s_tensors_cannot_be_exchanged(on_cpu):
    """Its calls go to the memory that it was made of."""
    s = cpu_store(n=8)
    for name in ("codes", "scale"):
        t = getattr(s, name)
        with pytest.raises(AttributeError):
            setattr(s, name, t.clone())
        assert getattr(s, name) is t
    s.codes[:] = 3       # what they hold can be
    assert addresses(s) == (s.codes.data_ptr(), s.scale.data_ptr()) and (s.codes == 3).all()


def test_kernels_do_not_spill():
    """The 256-column kernels stand close to the 256 registers that two waves to a SIMD leave."""
    from test_host_logic import test_scan_kernels_do_not_spill as check
    check("mx.hip", ["mx_ingest_kernel", "mx_append_kernel", "mx_gather_kernel", "mx_attn_kernel", "mx_merge_kernel"])
