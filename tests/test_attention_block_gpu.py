"""The attention layer as programs run it: steps captured beside eager calls of the same block, one block on several streams."""

import gc

import pytest
import torch

from dromos_b200 import abi, host
from tests import util
from tests.test_attention_layer_gpu import make_block, normal

pytestmark = pytest.mark.gpu

WIDTH, K, G, D, P = 256, 2, 4, 64, 16
PRODUCTS = pytest.mark.parametrize("wtype", [abi.W_BF16, abi.W_INT8, abi.W_FP8, abi.W_NVFP4], ids=["bf16", "int8", "fp8", "nvfp4"])


def int32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def decode_step(block, rows, page0, seed):
    """Sequences that hold three tokens each, on pages of their own from page0 on, and what a call for each one's next token takes."""
    table = torch.arange(page0, page0 + rows, dtype=torch.int32).reshape(rows, 1).cuda()
    three = host.KvBatch(int32([3 * i for i in range(rows + 1)]), int32([3] * rows), table, 3 * rows, 3)
    block(normal((3 * rows, WIDTH), seed).to(torch.bfloat16).cuda(), normal((3 * rows, WIDTH), seed + 1).cuda(), three)
    one = host.KvBatch(int32(list(range(rows + 1))), int32([4] * rows), table, rows, 1)
    return normal((rows, WIDTH), seed + 2).to(torch.bfloat16).cuda(), normal((rows, WIDTH), seed + 3).cuda(), one


@PRODUCTS
@pytest.mark.parametrize("rows", [9, 16, 64])
def test_a_captured_step_outlives_a_longer_prompt(lx, wtype, rows):
    """Replays of a captured step write to no memory but their own, whatever the same block is called for in between; a step that is
    computed again gives the same bits (its tokens are appended to the same slots)."""
    block, _, _ = make_block(lx, "fp8", D, K, G, WIDTH, P, 160, wtype=wtype)
    x, h, step = decode_step(block, rows, 0, 10)
    want = [t.clone() for t in block(x, h, step)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = block(x, h, step)
    n = 300
    prompt = host.KvBatch(int32([0, n]), int32([n]), torch.arange(100, 100 + n // P + 1, dtype=torch.int32)[None].cuda(), n, n)
    rows_in, residual = normal((n, WIDTH), 20).to(torch.bfloat16).cuda(), normal((n, WIDTH), 21).cuda()
    first = [t.clone() for t in block(rows_in, residual, prompt)]
    torch.cuda.synchronize()
    gc.collect()
    sizes = [lx.lx_gemm_workspace_bytes(m, k, 0) for m in (rows, 3 * rows, n) for k in (WIDTH, K * G * D)]
    others = [torch.full((size,), 0x5A, dtype=torch.uint8, device="cuda") for size in sizes for _ in range(8)]
    for _ in range(5):
        for t in got:
            t.zero_()
        graph.replay()
        again = block(rows_in, residual, prompt)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(again, first))
        assert all(bool((t == 0x5A).all()) for t in others)
    util.check_status(lx)


@PRODUCTS
def test_one_block_on_two_streams(lx, wtype):
    block, _, _ = make_block(lx, "int8", D, K, G, WIDTH, P, 100, wtype=wtype)
    steps = [decode_step(block, 16, 0, 30), decode_step(block, 64, 20, 40)]
    want = [[t.clone() for t in block(*s)] for s in steps]
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in steps], [[], []]
    for _ in range(50):
        for stream, step, out in zip(streams, steps, outs):
            with torch.cuda.stream(stream):
                out.append(block(*step))
    torch.cuda.synchronize()
    util.check_status(lx)
    for all_of, w in zip(outs, want):
        assert all(torch.equal(a, b) for out in all_of for a, b in zip(out, w))
