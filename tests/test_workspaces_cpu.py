"""Which device memory a layer of dromos_b200.host keeps between calls, seen without a GPU through a library that computes nothing.

A captured graph goes on using the workspace of the calls it holds. A layer that kept one workspace for all calls would hand the graph's
back to the allocator once a larger call came, and calls on two streams would prepare their activations in the same bytes. So a call takes
its workspace from torch's allocator and keeps nothing: what belongs to a graph is then in the graph's own pool."""

import types
import weakref

import pytest
import torch

from dromos_b200 import abi, host

WORKSPACES = {"lx_gemm_w": -2}  # where a call has its workspace's address


class Recorder:
    """Stands in for the library: calls succeed, and note which of the tensors made by the layer their workspace is."""

    def __init__(self, monkeypatch):
        self.made, self.seen = [], []
        empty = torch.empty

        def noted(*args, **kw):
            t = empty(*args, **kw)
            self.made.append((weakref.ref(t), t.data_ptr(), t.numel() * t.element_size()))
            return t

        monkeypatch.setattr(host.torch, "empty", noted)
        monkeypatch.setattr(host, "_raw_stream", lambda: 0)

    def lx_gemm_workspace_bytes(self, M, K, math):
        return 2 * M * K

    def call(self, name, args):
        at = args[WORKSPACES[name]]
        alive = [size for ref, address, size in self.made if ref() is not None and address == at]
        self.seen.append(alive)
        return 0

    def lx_gemm_w(self, *args):
        return self.call("lx_gemm_w", args)

    def kept(self, results):
        mine = {id(r) for r in results}
        return [size for ref, _, size in self.made if ref() is not None and id(ref()) not in mine]


def stored(wtype):
    return types.SimpleNamespace(wtype=wtype, ref=lambda: None)


@pytest.mark.parametrize("wtype", [abi.W_BF16, abi.W_INT8, abi.W_FP8, abi.W_NVFP4])
def test_a_product_keeps_no_workspace(monkeypatch, wtype):
    lib = Recorder(monkeypatch)
    layer = host.Linear(lib, stored(wtype), 32, 64)
    outs = [layer(torch.zeros((M, 64))) for M in (16, 200, 16, 9)]
    assert [max(sizes) >= 2 * M * 64 for sizes, M in zip(lib.seen, (16, 200, 16, 9))] == [True] * 4
    assert lib.kept(outs) == []
