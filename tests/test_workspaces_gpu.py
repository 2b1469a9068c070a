"""Routed experts captured in a graph beside larger calls of the same layer, and on two streams at once."""

import gc

import pytest
import torch

from dromos_b200 import abi, host
from tests import util

pytestmark = pytest.mark.gpu

E, L, I, TOP_K = 8, 512, 256, 2


def layer_and_inputs(lx, wtype, tokens):
    g = torch.Generator(device="cuda").manual_seed(1)
    gate_up, down = ((torch.randn(shape, generator=g, device="cuda") * 0.02).to(torch.bfloat16) for shape in ((E, 2 * I, L), (E, L, I)))
    layer = host.Experts(lx, host.store_weight(lx, gate_up, wtype), host.store_weight(lx, down, wtype), E, L, I, TOP_K)
    inputs = []
    for T in tokens:
        latent = torch.randn((T, L), generator=g, device="cuda").to(torch.bfloat16)
        inputs.append((latent, *layer.route(torch.randn((T, E), generator=g, device="cuda"))))
    return layer, inputs


@pytest.mark.parametrize("wtype", [abi.W_BF16, abi.W_INT8, abi.W_FP8], ids=["bf16", "int8", "fp8"])
def test_captured_experts_outlive_a_larger_call(lx, wtype):
    layer, (few, many) = layer_and_inputs(lx, wtype, (12, 500))
    want, large = layer(*few).clone(), layer(*many).clone()
    graph = torch.cuda.CUDAGraph()
    layer(*few)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = layer(*few)
    assert torch.equal(layer(*many), large)
    torch.cuda.synchronize()
    gc.collect()
    sizes = [lx.lx_moe_grouped_workspace_bytes(T, L, I, E, TOP_K, 0) for T in (12, 500)]
    others = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for size in sizes for _ in range(8)]
    for _ in range(5):
        got.zero_()
        graph.replay()
        again = layer(*many)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(again, large) and all(bool((t == 0x5A).all()) for t in others)
    util.check_status(lx)


def test_experts_on_two_streams(lx):
    layer, inputs = layer_and_inputs(lx, abi.W_FP8, (12, 40))
    want = [layer(*x).clone() for x in inputs]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in inputs], [[], []]
    for _ in range(50):
        for stream, x, out in zip(streams, inputs, outs):
            with torch.cuda.stream(stream):
                out.append(layer(*x))
    torch.cuda.synchronize()
    util.check_status(lx)
    for all_of, w in zip(outs, want):
        assert all(torch.equal(o, w) for o in all_of)
