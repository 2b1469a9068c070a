"""Which device memory a layer of dromos_b200.host keeps between calls, seen without a GPU through a library that computes nothing.

A captured graph goes on using the workspace of the calls it holds. A layer that kept one workspace for all calls would hand the graph's
back to the allocator once a larger call came, and calls on two streams would prepare their activations in the same bytes. So a call takes
its workspace from torch's allocator and keeps nothing: what belongs to a graph is then in the graph's own pool."""

import types
import weakref

import pytest
import torch

from dromos_b200 import abi, host

WORKSPACES = {"lx_gemm_w": -2, "lx_moe_experts_grouped": 7, "lx_b200_linear_allgather": -3}  # where a call has its workspace's address


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

    def lx_moe_grouped_workspace_bytes(self, T, L, I, E, top_k, math):
        return 64 * T * L

    def call(self, name, args):
        at = args[WORKSPACES[name]]
        at = getattr(at, "value", at)
        alive = [size for ref, address, size in self.made if ref() is not None and address == at]
        self.seen.append(alive)
        return 0

    def lx_gemm_w(self, *args):
        return self.call("lx_gemm_w", args)

    def lx_moe_experts_grouped(self, *args):
        return self.call("lx_moe_experts_grouped", args)

    def lx_b200_linear_allgather(self, *args):
        return self.call("lx_b200_linear_allgather", args)

    def lx_b200_wait_arrivals(self, *args):
        return 0

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


def test_routed_experts_keep_no_workspace(monkeypatch):
    lib = Recorder(monkeypatch)
    layer = host.Experts(lib, stored(abi.W_FP8), stored(abi.W_FP8), 8, 64, 32, 2)
    outs = []
    for T in (9, 100, 9, 33):
        outs.append(layer(torch.zeros((T, 64)), torch.zeros((T, 2), dtype=torch.int32), torch.zeros((T, 2))))
        assert max(lib.seen[-1]) >= 64 * T * 64
    assert lib.kept(outs) == []


def test_a_product_gathered_over_ranks_keeps_no_workspace(monkeypatch):
    lib = Recorder(monkeypatch)
    monkeypatch.setattr(host, "_stream", lambda: None)
    layer = object.__new__(host.FusedShardedLinear)  # without the buffers that ranks exchange
    layer.lib, layer.world, layer.rank, layer.N, layer.K, layer.n0, layer.n1, layer.max_rows = lib, 1, 0, 32, 64, 0, 32, 256
    layer.weight, layer.y = stored(abi.W_FP8), torch.zeros((2, 256, 32))
    layer._y_ptrs, layer._c_ptrs, layer._c_array, layer._calls, layer._total = [0], [0], None, 0, {16: 1, 200: 1}
    for M in (16, 200, 16):
        layer(torch.zeros((M, 64)))
        assert max(lib.seen[-1]) >= 2 * M * 64
    assert lib.kept([]) == []
