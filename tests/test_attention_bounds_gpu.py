"""Batches at the ends of what their arrays can say: windows and lengths near 2^31, rows that cannot be, more sequences and row blocks than
the kernels look at in one round. Tolerances are those of test_attention_layer_gpu."""

import math

import pytest
import torch

from dromos_b200 import host
from tests import kv_reference as R
from tests import util
from tests.test_attention_layer_gpu import check_attention, make_cache, normal, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [2**31 - 1, 2**31 - 7, 2**30])
@pytest.mark.parametrize("n,length", [(8, 3), (8, 7), (200, 100), (200, 1)])
def test_the_widest_windows_over_sequences_shorter_than_their_new_tokens(lx, n, length, window):
    """Slots before the first see nothing, the others all that is there: as without a window."""
    S = R.Sequences([n, 1], [n, 20], 16, seed=7)
    cache, _ = make_cache(lx, S, 1, 64, "fp8", 50)
    q = normal((S.rows, 4 * 64), 51, dtype=torch.bfloat16).cuda()
    want = host.Attention(cache, 4)(put(S, lengths=[length, 20]), q)
    got = host.Attention(cache, 4, window=window)(put(S, lengths=[length, 20]), q)
    util.check_status(lx)
    assert torch.equal(got, want) and bool((want[:n - length] == 0).all()) and bool((want[n - length:n] != 0).any(1).all())


@pytest.mark.parametrize("n", [1, 9, 200])
@pytest.mark.parametrize("length", [2**31 - 1, 2**31 - 40, 2**31 - 128, 2**31 - 129])
def test_lengths_up_to_the_largest(lx, n, length):
    """No page holds such slots: the rows are not-a-number and it is reported, the sequence beside them is as it is alone."""
    S = R.Sequences([n, 3], [n + 40, 50], 16, seed=9)
    cache, _ = make_cache(lx, S, 2, 64, "int8", 60)
    q = normal((S.rows, 4 * 64), 61, dtype=torch.bfloat16).cuda()
    attend = host.Attention(cache, 4, window=50)
    right = attend(put(S), q)
    util.check_status(lx)
    out = attend(put(S, lengths=[length, 50]), q)
    torch.cuda.synchronize()
    assert lx.lx_b200_last_error() == 9
    assert bool(out[:n].isnan().all())
    assert torch.equal(out[n:], right[n:])


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("P", [16, 128])
def test_queries_of_slots_up_to_the_largest_are_turned(lx, n, P):
    K, D = 1, 64
    S = R.Sequences([n, 2], [n, 9], P, seed=10)
    cache, (k0, ks0, v0, vs0) = make_cache(lx, S, K, D, "fp8", 70)
    x, q = normal((S.rows, K * D), 71).cuda(), normal((S.rows, 2 * D), 72).cuda()
    length, rotary = 2**31 - 1, host.Rotary.of(D, device="cuda")
    positions = torch.tensor(list(range(length - n, length)) + [7, 8], dtype=torch.int32)
    frequencies = rotary.frequencies.cpu()
    out = torch.full((S.rows, 2 * D), 7.5, device="cuda")
    cache.append(put(S, lengths=[length, 9]), x, x, q=q, rotary=rotary, q_out=out)
    torch.cuda.synchronize()
    assert lx.lx_b200_last_error() == 9  # their pages are not there
    want = R.rotate(q.cpu().double().reshape(S.rows, 2, D), positions, frequencies, False)
    size = R.rotate(q.cpu().double().abs().reshape(S.rows, 2, D), torch.zeros_like(positions), frequencies, False)
    size = (size[..., :D // 2] + size[..., D // 2:]).repeat(1, 1, 2)
    # 2^-21 of the pair, and the digits of an angle of 2^31 radians in 64 bits: in the kernel a product, the constant that makes it turns and
    # their product (2.5 roundings of 2^-53), here one product; 3.5 x 2^31 x 2^-53 is below 2^-20
    assert bool(((out.cpu().double().reshape(S.rows, 2, D) - want).abs() <= size * (2.0**-21 + 2.0**-20)).all())
    v, vs = R.append(v0, vs0, "fp8", x.cpu().double()[:, None], S.starts, [length, 9], S.table, P)
    assert torch.equal(cache.v.cpu(), v) and torch.equal(cache.v_scale.cpu(), vs)
