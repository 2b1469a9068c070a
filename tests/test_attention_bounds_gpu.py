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


def attend_over(S, attend, q, starts, lengths):
    out = torch.full_like(q, 9.5)
    attend(put(S, starts=starts, lengths=lengths), q, out=out)
    torch.cuda.synchronize()
    return out


# starts that cannot be (rows before, past and against the buffer's), and a batch in whose place the sequences concerned have no new tokens
@pytest.mark.parametrize("n", [1, 20, 200])
@pytest.mark.parametrize("bad,clean", [((0, 2, 4, None, 10**6), (0, 2, 4, None, None)), ((0, 2, 4, None, 2**31 - 1), (0, 2, 4, None, None)), ((-3, 2, 4, None, -1), (2, 2, 4, None, -1)),
                                       ((-2**31, 2, 4, None, -1), (2, 2, 4, None, -1)), ((4, 2, 4, None, -1), (2, 2, 4, None, -1)),
                                       ((0, 2, 4, None, 3), (0, 2, 4, None, None))])
def test_attention_leaves_alone_rows_that_cannot_be(lx, n, bad, clean):
    """They are reported; the other sequences' rows have the bits of a batch without them, other rows stay as they are."""
    S = R.Sequences([2, 2, n, 2], [20, 33, n + 60, 40], 16, seed=2)
    cache, _ = make_cache(lx, S, 2, 64, "fp8", 11)
    q, attend = normal((S.rows, 8 * 64), 12, dtype=torch.bfloat16).cuda(), host.Attention(cache, 8)
    name = {None: 4 + n, -1: S.rows}
    bad, clean = ([name.get(x, x) for x in s] for s in (bad, clean))
    want = attend_over(S, attend, q, clean, S.total)
    assert lx.lx_b200_last_error() == 0
    got = attend_over(S, attend, q, bad, S.total)
    assert lx.lx_b200_last_error() == 9
    assert torch.equal(got, want)
    row = torch.zeros(S.rows, dtype=torch.bool)
    for a, b in zip(clean, clean[1:]):
        row[a:b] = True
    assert bool((got.cpu()[~row] == 9.5).all()) and bool((got.cpu()[row] != 9.5).any(1).all())


@pytest.mark.parametrize("n,sequences", [(200, 40), (200, 700), (3, 300)])
def test_attention_of_sequences_that_share_their_rows(lx, n, sequences):
    """More row blocks than the rows there are could have, which the order of work has room for: reported, as descending rows are. Each
    sequence reads the same keys, so whichever writes a row last writes the same value, to the rounding of parts joined in another order."""
    K, G, D, P, length = 1, 4, 64, 16, n + 30
    S = R.Sequences([n], [length], P, seed=4, rows_behind=2)
    cache, (k, ks, v, vs) = make_cache(lx, S, K, D, "fp8", 21)
    q, attend = normal((S.rows, G * D), 22, dtype=torch.bfloat16), host.Attention(cache, G)
    batch = host.KvBatch(torch.tensor([0, n] * sequences, dtype=torch.int32).cuda(), torch.full((2 * sequences - 1,), length, dtype=torch.int32).cuda(),
                         S.matrix.repeat(2 * sequences - 1, 1).cuda(), S.rows, n)
    out = torch.full((S.rows, G * D), 9.5, dtype=torch.bfloat16, device="cuda")
    attend(batch, q.cuda(), out=out)
    torch.cuda.synchronize()
    assert lx.lx_b200_last_error() == 9
    want, size = R.attention(q.double(), k, ks, v, vs, "fp8", S.starts, S.total, S.table, P, G, attend.scale, 0)
    kmax = (R.decode(k, "fp8").abs() * ks.double()[:, :, None, None]).amax((0, 2))[0]
    d = attend.scale * (q.double().reshape(S.rows, G, D).abs() * kmax).sum(2, keepdim=True) * 2.0**-24 * D
    bound = want.abs() * 2.0**-8 + size * (2.0**-10 + 2 * d.expand(-1, -1, D).reshape(S.rows, -1)) + 1e-30
    bound += (size.reshape(S.rows, G, D).amax(2, keepdim=True) * 2.0**-31 * length).expand(-1, -1, D).reshape(S.rows, -1)
    assert bool(((out.cpu().double() - want).abs() <= bound)[:n].all()) and bool((out[n:] == 9.5).all())


def test_attention_of_more_sequences_than_a_round_of_the_plan(lx):
    """1300 sequences, some for either kernel, many in the second round of 1024."""
    g = torch.Generator().manual_seed(31)
    total = torch.randint(1, 90, (1300,), generator=g).tolist()
    new = [0 if i % 7 == 3 else min(t, 30) if i % 40 == 0 else 1 for i, t in enumerate(total)]
    S = R.Sequences(new, total, 16, seed=32, rows_behind=1)
    check_attention(lx, S, 1, 4, 64, "int8")


@pytest.mark.parametrize("D,G,n", [(64, 64, 100), (256, 33, 100)])
def test_attention_of_more_row_blocks_than_a_round_of_the_plan(lx, D, G, n):
    """More than 1024 blocks of 256 rows (128 with 256 values per head), most sequences' last ones partly full."""
    rows = 128 if D == 256 else 256
    sequences = 1024 // (n * G // rows) + 2
    S = R.Sequences([n] * sequences, [n + 3 + i for i in range(sequences)], 32, seed=33)
    assert sum(-(-m * G // rows) for m in S.new) > 1024
    check_attention(lx, S, 1, G, D, "fp8")
