"""The attention layer as programs run it: steps captured beside eager calls of the same block, one block on several streams."""

import gc

import pytest
import torch

from dromos_b200 import abi, host
from tests import kv_reference as R
from tests import util
from tests.test_attention_layer_gpu import make_block, make_cache, normal, put

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


def poison(mib=256):
    """What the allocator hands out next holds not-a-number."""
    blocks = [torch.full((n,), float("nan"), device="cuda") for n in [mib * 2**18] + [2**e for e in range(8, 21) for _ in range(4)]]
    torch.cuda.synchronize()
    del blocks


# G, new tokens, hint: few rows, tiles beside few rows, tiles alone (a group of more heads than the kernel for few rows takes), no tokens at all
PADDED = pytest.mark.parametrize("group,new,behind", [(4, [1, 1, 1], 2), (4, [1] * 20, 12), (4, [60, 1, 0, 7], 5), (40, [3, 1], 3), (4, [0, 0], 4), (4, [], 3), (4, [130], 1000)])


@PADDED
def test_rows_behind_the_last_sequence_are_zero_where_the_library_makes_the_results(lx, group, new, behind):
    K, D, P = 2, 64, 16
    S = R.Sequences(new, [n + 5 for n in new], P, seed=3, rows_behind=behind)
    cache, _ = make_cache(lx, S, K, D, "fp8", 5)
    q, attend = normal((S.rows, K * group * D), 6, dtype=torch.bfloat16).cuda(), host.Attention(cache, K * group)
    poison()
    out = attend(put(S), q)
    util.check_status(lx)
    assert bool((out[S.tokens:] == 0).all()) and bool(out.isfinite().all())
    own = torch.full_like(out, 9.5)
    assert attend(put(S), q, out=own) is own and torch.equal(own[:S.tokens], out[:S.tokens]) and bool((own[S.tokens:] == 9.5).all())


@pytest.mark.parametrize("rows,behind", [(3, 2), (12, 4), (20, 44), (0, 6)])
@pytest.mark.parametrize("wtype", [abi.W_BF16, abi.W_NVFP4], ids=["bf16", "nvfp4"])
def test_a_padded_step(lx, rows, behind, wtype):
    """A step of a fixed count of rows of which the last ones belong to no sequence: these get nothing from the block, whatever is in memory."""
    block, _, _ = make_block(lx, "fp8", D, K, G, WIDTH, P, 100, wtype=wtype)
    if rows:
        decode_step(block, rows, 0, 50)
    table = torch.arange(rows, dtype=torch.int32).reshape(rows, 1).cuda()
    batch = host.KvBatch(int32(list(range(rows + 1))), int32([4] * rows), table, rows + behind, 1)
    x, h = normal((rows + behind, WIDTH), 60).to(torch.bfloat16).cuda(), normal((rows + behind, WIDTH), 61).cuda()
    poison()
    got_h, got_x = block(x, h, batch)
    util.check_status(lx)
    want_h, want_x = block.norm(None, h[rows:])
    assert torch.equal(got_h[rows:], want_h) and torch.equal(got_x[rows:], want_x)
    assert bool(got_h.isfinite().all()) and bool(got_x.isfinite().all())


@pytest.mark.parametrize("new", [1, 4, 24])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_attention_right_behind_appends_to_what_it_reads(lx, kind, new):
    """Steps back to back on one stream, whose kernels may be resident before the last one has ended, and with a wait between any two calls:
    the same codes, scales and results. Louder and louder tokens, so that appends rewrite the codes that the step before has read."""
    S, steps, heads = 8, 30, K * G
    table = torch.randperm(8 * 48, generator=torch.Generator().manual_seed(3)).to(torch.int32).reshape(8, 48).cuda()
    starts, T = int32([new * i for i in range(S + 1)]), S * new
    rows = [(normal((T, (heads + 2 * K) * D), 100 + i) * 1.2**i).cuda() for i in range(steps)]
    lengths = [int32([new * (i + 1) + s for s in range(S)]) for i in range(steps)]
    results = []
    for wait in (False, True):
        cache = host.KvCache.empty(lx, {"fp8": abi.W_FP8, "int8": abi.W_INT8}[kind], 8 * 48, K, D, P)
        attend, turn, outs = host.Attention(cache, heads), host.Rotary.of(D, device="cuda"), []
        torch.cuda.synchronize()
        for i in range(steps):
            batch, x = host.KvBatch(starts, lengths[i], table, T, new), rows[i]
            q = cache.append(batch, x[:, heads * D:(heads + K) * D], x[:, (heads + K) * D:], q=x[:, :heads * D], rotary=turn)
            if wait:
                torch.cuda.synchronize()
            outs.append(attend(batch, q))
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        util.check_status(lx)
        results.append([torch.stack(outs), cache.k, cache.v, cache.k_scale, cache.v_scale])
    assert all(torch.equal(a, b) for a, b in zip(*results)) and bool(results[0][0].isfinite().all())
