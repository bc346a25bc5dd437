"""Stores and caches of the block-scaled kind without a GPU: copies, and calls that are refused before anything is launched."""
import copy
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
