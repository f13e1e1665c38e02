"""Device memory lives as long as anything of the binding that points into it."""
import gc
import weakref

import numpy as np
import pytest

from cudabackend_b200 import api


@pytest.fixture
def destroyed(monkeypatch):
    """Handles whose memory was destroyed; the library is replaced by one that hands out addresses and frees nothing."""
    handles = []

    def call(name, *args):
        if name == "cudaGetMemoryPointer":
            args[1]._obj.value = 0x1000 * args[0]
        elif name == "cudaCreateMemoryView":
            args[0]._obj.value = 100 + args[3]
        elif name == "cudaDestroyMemoryDescriptor":
            handles.append(args[0])

    monkeypatch.setattr(api, "call", call)
    yield handles
    gc.collect()


def test_an_address_keeps_its_memory(destroyed):
    address = api.Memory(64, handle=7).pointer()
    gc.collect()
    assert destroyed == [] and address == 0x7000 and isinstance(address, int)
    inside = address + 16
    del address
    gc.collect()
    assert destroyed == [] and inside == 0x7010
    del inside
    gc.collect()
    assert destroyed == [7]


def test_an_address_is_a_number_like_any_other(destroyed):
    import ctypes
    import pickle
    address = api.Memory(64, handle=7).pointer()
    assert ctypes.c_void_p(address).value == 0x7000 and "%#x" % address == "0x7000" and {address: 1}[0x7000] == 1
    assert address - 0x6000 == 0x1000 and 16 + address == 0x7010 and address + 0.5 == 28672.5
    inside = address + np.int64(8)
    assert inside.memory is address.memory and inside == 0x7008
    copy = pickle.loads(pickle.dumps(address))
    assert type(copy) is int and copy == 0x7000


def test_destroy_frees_whoever_holds_the_address(destroyed):
    memory = api.Memory(64, handle=7)
    address = memory.pointer()
    memory.destroy()
    assert destroyed == [7]
    del memory, address
    gc.collect()
    assert destroyed == [7]


def test_a_view_keeps_the_memory_it_looks_into(destroyed):
    view = api.Memory(64, handle=7).view(32, 8)
    inner = view.view(8, 4)
    del view
    gc.collect()
    assert destroyed == []
    del inner
    gc.collect()
    assert sorted(destroyed) == [7, 104, 108]


@pytest.mark.gpu
def test_a_torch_tensor_over_the_memory_outlives_the_tensor_it_came_from(ctx):
    import torch

    class Holder:
        pass

    block = api.DeviceTensor((333, 2056), "float32")
    values = np.random.default_rng(111).normal(0, 1, block.shape).astype(np.float32)
    block.upload(ctx, values)
    ctx.synchronize()
    holder = Holder()
    holder.__cuda_array_interface__ = {"shape": block.shape, "typestr": "<f4", "data": (block.mem.pointer(), False), "version": 3}
    view = torch.as_tensor(holder, device="cuda")[1:]
    memory = weakref.ref(block.mem)
    del block, holder
    gc.collect()
    assert memory() is not None  # nothing is read before this is known
    assert np.array_equal(view.cpu().numpy(), values[1:])
