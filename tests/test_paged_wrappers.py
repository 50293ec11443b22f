"""What the wrappers of the paged operators hold and ask while they call, without a device: tensors
that say they are on one, and a library that only looks."""
import weakref

import pytest
import torch

from channel_b200 import paged


class OnDevice(torch.Tensor):
    """A host tensor that says it is on a CUDA device."""
    index = 0
    made = []

    def get_device(self):
        return self.index

    def new_empty(self, *size, **kw):
        t = torch.empty(*size, **kw)
        OnDevice.made.append(weakref.ref(t))
        return t


def placed(*shape, dtype=torch.float16):
    return torch.zeros(shape, dtype=dtype).as_subclass(OnDevice)


def chunk_call():
    qkv = placed(5, 8, 64)
    return paged.prompt_attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], placed(2, dtype=torch.int32), out=placed(5, 4, 64))


def prefix_call():
    pool = placed(3, 16, 2, 64)
    return paged.prefix_attention(placed(2, 4, 64), pool, pool, placed(2, 1, dtype=torch.int32), placed(2, dtype=torch.int32),
                                  out=placed(2, 4, 64))


class Library:
    """Calls that succeed; `seen` gets what `look` says at each."""
    def __init__(self, look):
        self.look, self.seen = look, {}

    def __getattr__(self, name):
        def call(*args):
            self.seen[name] = self.look()
            return 1024 if name.endswith("workspace") else 0
        return call


@pytest.fixture
def library(monkeypatch):
    def make(look):
        lib = Library(look)
        monkeypatch.setattr(paged.L, "load", lambda: lib)
        monkeypatch.setattr(paged, "_stream_of", lambda at: 0)
        OnDevice.made.clear()
        return lib
    return make


@pytest.mark.parametrize("call,name", [(chunk_call, "ch_chunk_attention"), (prefix_call, "ch_prefix_attention")])
def test_the_workspace_lives_until_the_call_returns(call, name, library, monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    lib = library(lambda: [t() is not None for t in OnDevice.made])
    call()
    assert lib.seen[name] == [True]


@pytest.mark.parametrize("call,name", [(chunk_call, "ch_chunk_attention"), (prefix_call, "ch_prefix_attention")])
def test_the_workspace_is_that_of_the_tensors_device(call, name, library, monkeypatch):
    current = [0]

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *why):
            current[0] = self.before

    monkeypatch.setattr(OnDevice, "index", 1)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    lib = library(lambda: current[0])
    call()
    assert lib.seen == {f"{name}_workspace": 1, name: 1} and current == [0]
