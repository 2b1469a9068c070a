"""Appending to the paged 8-bit cache, attention over it and the norms around a block, on the GPU against plain 64-bit
implementations, and a run of them together.

Tolerances, derived from the roundings of each operator:
  append     scales and the codes of values that no arithmetic touches (V; K where nothing turns) are equal bit for bit. A rotated
             value carries an error of 2^-21 of its pair's magnitude (sine, cosine, two products and a sum in f32, 2^-24 each, and the
             angle's rounding to f32, 2^-24 * pi), so its code may be that of a value so far off.
  queries    the same 2^-21, and their rounding to bf16, 2^-8 of the value (f32: none).
  attention  the rounding of the result to bf16, 2^-8 |o|; the weights' rounding to f16, 2^-11 of sum w |v|, and as much again for f32
             sums and exponentials; weights are scaled so that the largest w v-scale is 2^7 or more, so those below f16's normal
             range are off by 2^-32 of it at most (half of 2^-24); with codes of up to 448 (or 127) whose largest is at least half of that
             in every page a key adds 2^-32 max(w v-scale top), and max(w v-scale top) <= 2 max over the dims of sum w |v|:
             n 2^-31 of that in all; scores that are off by d move every weight by a factor within
             1 +- 2 d: d = |scale| sum |q k| (2^-11 for queries in f32, which are rounded to f16; D 2^-24 for the sum).
  norm       mean squares of positive terms 2^-19 (at most 32 + 10 additions in a chain, 2^-24 each), halved by the root; some
             more factors of 2^-24: 2^-19 of a term in all; bf16 results 2^-8 more.
"""

import math

import pytest
import torch

from dromos_b200 import abi, host
from tests import kv_reference as R
from tests import util

pytestmark = pytest.mark.gpu

WTYPE = {"fp8": abi.W_FP8, "int8": abi.W_INT8}


def normal(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def put(S: R.Sequences, lengths=None, starts=None, max_new=None):
    return host.KvBatch(torch.tensor(starts or S.starts, dtype=torch.int32).cuda(), torch.tensor(lengths or S.total, dtype=torch.int32).cuda(), S.matrix.cuda(),
                        tokens=S.rows, max_new=max(S.new + [0]) if max_new is None else max_new)


def make_cache(lx, S, heads, D, kind, seed):
    k, ks = R.stored(S.pages, heads, S.P, D, kind, seed)
    v, vs = R.stored(S.pages, heads, S.P, D, kind, seed + 1)
    return host.KvCache(lx, WTYPE[kind], k.cuda(), v.cuda(), ks.cuda(), vs.cuda()), (k, ks, v, vs)


# ---- append ------------------------------------------------------------------------------------------------------------------
def check_codes(got, want, values, slack, kind, what):
    """Codes equal, or those of a value within `slack` of the exact one (values and slack already divided by the scale)."""
    same = got == want
    lo, hi = R.decode(R.encode(values - slack, kind), kind), R.decode(R.encode(values + slack, kind), kind)
    have = R.decode(got, kind)
    assert bool((same | ((have >= lo) & (have <= hi))).all()), what


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("D,P,rotary,interleaved,dtype,q_out", [
    (64, 16, 64, False, torch.float32, torch.bfloat16), (128, 64, 128, False, torch.bfloat16, torch.bfloat16), (128, 16, 64, True, torch.float32, torch.float32),
    (256, 32, 256, True, torch.bfloat16, torch.bfloat16), (256, 128, 8, False, torch.float32, torch.bfloat16), (128, 32, 0, False, torch.float32, torch.bfloat16),
    (64, 128, 24, True, torch.bfloat16, torch.float32)])
def test_append(lx, kind, D, P, rotary, interleaved, dtype, q_out):
    K, H = 2, 6
    S = R.Sequences([1, 0, 2 * P + 3, P, 5, 1, 1], [1, 4, 3 * P + 1, P, 2 * P + 2, 3 * P, 2 * P + 1], P, seed=D + P, rows_behind=2)
    cache, (k0, ks0, v0, vs0) = make_cache(lx, S, K, D, kind, 5)
    rows = normal((S.rows, (H + 2 * K) * D), 7, 3.0, dtype)
    rows[S.starts[4]] *= 40  # a loud token: the page's scale grows, what it holds is rounded to it
    positions = S.slots() + 900000
    frequencies = torch.pow(torch.tensor(10000.0, dtype=torch.float64), -torch.arange(0, rotary, 2).double() / max(rotary, 1)) if rotary else None
    dev = rows.cuda()
    out = torch.full((S.rows, H * D), 7.5, dtype=q_out, device="cuda")
    got = cache.append(put(S), dev[:, H * D:(H + K) * D], dev[:, (H + K) * D:], q=dev[:, :H * D], rotary=host.Rotary(frequencies.cuda(), interleaved) if rotary else None,
                       positions=positions.cuda(), q_out=out)
    util.check_status(lx)
    assert got is out
    x = rows.double().reshape(S.rows, H + 2 * K, D)
    turned = R.rotate(x[:, :H + K], positions, frequencies, interleaved)
    pair = R.rotate(x[:, :H + K].abs(), torch.zeros_like(positions), frequencies, interleaved)  # the magnitudes
    if rotary:
        first, second = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
        pair[..., first] = pair[..., second] = pair[..., first] + pair[..., second]
    slack = pair * 2.0**-21 if rotary else torch.zeros_like(pair)
    q = out.cpu().double().reshape(S.rows, H, D)
    assert bool((q[S.tokens:] == 7.5).all()), "rows behind the last sequence are left as they were"
    bound = slack[:, :H] + turned[:, :H].abs() * (2.0**-8 if q_out == torch.bfloat16 else 2.0**-24)
    assert bool(((q - turned[:, :H]).abs() <= bound)[:S.tokens].all())
    v, vs = R.append(v0, vs0, kind, x[:, H + K:], S.starts, S.total, S.table, P)
    assert torch.equal(cache.v_scale.cpu(), vs) and torch.equal(cache.v.cpu(), v)
    k, ks = R.append(k0, ks0, kind, turned[:, H:], S.starts, S.total, S.table, P)
    assert torch.equal(cache.k_scale.cpu(), ks)
    have = cache.k.cpu()
    if not rotary:
        assert torch.equal(have, k)
    touched = torch.zeros_like(k, dtype=torch.bool)
    row = 0
    for s, (n, t) in enumerate(zip(S.new, S.total)):
        for slot in range(t - n, t):
            p, o = S.table[s][slot // P], slot % P
            check_codes(have[p, :, o], k[p, :, o], turned[row, H:] / ks[p].double()[:, None], slack[row, H:] / ks[p].double()[:, None], kind, (s, slot))
            touched[p, :, o] = True
            row += 1
    assert torch.equal(have[~touched], k[~touched])


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_append_token_by_token(lx, kind):
    """Single tokens into fresh pages: scales start anew at a page's first slot and grow with what comes; positions default to slots."""
    K, D, P = 1, 64, 16
    cache = host.KvCache.empty(lx, WTYPE[kind], 4, K, D, P)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda()
    starts, lengths = torch.tensor([0, 1], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    batch = host.KvBatch(starts, lengths, table, tokens=1, max_new=1)
    k, ks = cache.k.cpu(), cache.k_scale.cpu()
    v, vs = cache.v.cpu(), cache.v_scale.cpu()
    for i in range(35):
        x = normal((1, D), 100 + i, 2.0 ** ((i * 5) % 7 - 3))
        lengths.fill_(i + 1)
        assert cache.append(batch, x.cuda(), x.cuda()) is None
        k, ks = R.append(k, ks, kind, x.double()[:, None], [0, 1], [i + 1], [[2, 0, 3]], P)
        v, vs = R.append(v, vs, kind, x.double()[:, None], [0, 1], [i + 1], [[2, 0, 3]], P)
        assert torch.equal(cache.k_scale.cpu(), ks) and torch.equal(cache.k.cpu(), k) and torch.equal(cache.v.cpu(), v), i
    util.check_status(lx)
    one = host.Rotary.of(D, device="cuda")
    q = normal((1, D), 3)
    lengths.fill_(36)
    a = cache.append(batch, x.cuda(), x.cuda(), q=q.cuda(), rotary=one)
    b = cache.append(batch, x.cuda(), x.cuda(), q=q.cuda(), rotary=one, positions=torch.tensor([35], dtype=torch.int32).cuda())
    assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_append_of_zeros_extremes_and_values_that_are_not_finite(lx, kind):
    K, D, P = 3, 128, 32
    S = R.Sequences([3, 3, 3, 3], [3, P + 3, P + 5, 2 * P + 1], P, seed=1)
    cache, (k0, ks0, v0, vs0) = make_cache(lx, S, K, D, kind, 9)
    x = normal((S.rows, K * D), 4).reshape(S.rows, K, D)
    x[0:3] = 0
    x[1, 0, 0] = -0.0
    x[3:6, 0] = 3e38
    x[3:6, 1] = 1e-40
    x[3:6, 2] = 2.0**-93
    x[6, 0, 5], x[7, 1, 9], x[8, 2, 127] = math.nan, math.inf, -math.inf
    top = R.TOP[kind]
    x[9, 0, 0], x[9, 1, 0], x[9, 2, 0] = top, top * (1 + 2.0**-22), top * 2.0**20
    dev = x.reshape(S.rows, -1).cuda()
    cache.append(put(S), dev, dev)
    util.check_status(lx)
    v, vs = R.append(v0, vs0, kind, x.double(), S.starts, S.total, S.table, P)
    k, ks = R.append(k0, ks0, kind, x.double(), S.starts, S.total, S.table, P)
    for got, want in ((cache.v_scale, vs), (cache.k_scale, ks)):
        assert torch.equal(got.cpu().nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
    assert int(vs.isnan().sum()) == 3
    assert torch.equal(R.decode(cache.v.cpu(), kind), R.decode(v, kind)) and torch.equal(R.decode(cache.k.cpu(), kind), R.decode(k, kind))


def test_append_leaves_alone_what_cannot_be(lx):
    """A sequence shorter than its new tokens, rows outside the buffers and pages outside the cache are not written and are reported; the
    sequences beside them are appended. The kernel's own checks answer: nothing is read or written out of range."""
    K, D, P, kind = 1, 64, 16, "fp8"
    S = R.Sequences([2, 2, 20, 2], [P, P, 20, P], P, seed=2)
    cache, (k0, ks0, v0, vs0) = make_cache(lx, S, K, D, kind, 11)
    x = normal((S.rows, D), 5)
    dev = x.cuda()
    S.table[2][1] = S.pages  # one past the cache
    S.matrix[2, 1] = S.pages
    lengths = [S.total[0], 1, S.total[2], S.total[3]]
    cache.append(put(S, lengths=lengths), dev, dev)
    torch.cuda.synchronize()
    assert lx.lx_b200_last_error() == 9 and lx.lx_b200_last_error() == 0
    v, vs = R.append(v0, vs0, kind, x.double()[:, None], S.starts, lengths, S.table, P)
    assert torch.equal(cache.v.cpu(), v) and torch.equal(cache.v_scale.cpu(), vs)
    # rows past the buffers, descending rows
    for starts in ([0, 2, 4, 24, 10**6], [0, 5, 4, 24, 26], [-3, 2, 4, 24, 26]):
        cache, (k0, ks0, v0, vs0) = make_cache(lx, S, K, D, kind, 11)
        lengths = [max(t, b - a) if 0 <= b - a < 10**5 else t for t, a, b in zip(S.total, starts, starts[1:])]
        cache.append(put(S, starts=starts, lengths=lengths), dev, dev)
        torch.cuda.synchronize()
        assert lx.lx_b200_last_error() == 9
        v, vs = R.append(v0, vs0, kind, x.double()[:, None], starts, lengths, S.table, P)
        assert torch.equal(cache.v.cpu(), v) and torch.equal(cache.v_scale.cpu(), vs), starts


def test_append_of_more_tokens_than_the_hint(lx):
    K, D, P, kind = 2, 64, 16, "int8"
    S = R.Sequences([70, 3], [75, 9], P, seed=3)
    x = normal((S.rows, K * D), 6)
    results = []
    for hint in (1, 70, 0, 10**6):  # both ways of cutting the work
        cache, _ = make_cache(lx, S, K, D, kind, 13)
        cache.append(put(S, max_new=hint), x.cuda(), x.cuda())
        results.append(torch.cat([cache.k.flatten(), cache.v.flatten(), cache.k_scale.flatten().view(torch.uint8)]).cpu())
    util.check_status(lx)
    assert all(torch.equal(r, results[0]) for r in results)


# ---- attention ---------------------------------------------------------------------------------------------------------------
def check_attention(lx, S, K, G, D, kind, window=0, dtype=torch.bfloat16, seed=0, scale=None, spread=1.0, wreck=None, max_new=None, cache=None):
    H = K * G
    cache, (k, ks, v, vs) = cache or make_cache(lx, S, K, D, kind, 20 + seed)
    q = normal((S.rows, H * D + 8), 30 + seed, spread, dtype)
    dev = q.cuda()[:, :H * D]  # a row stride of its own
    out = torch.full((S.rows, H * D + 16), 9.5, dtype=torch.bfloat16, device="cuda")
    attend = host.Attention(cache, H, scale=scale, window=window)
    batch = put(S, max_new=max_new)
    got = attend(batch, dev, out=out[:, :H * D])
    util.check_status(lx)
    again = attend(batch, dev)
    assert torch.equal(got[:S.tokens], again[:S.tokens]), "the same bits every time"
    assert bool((out[S.tokens:] == 9.5).all()) and bool((out[:, H * D:] == 9.5).all())
    qd = q[:, :H * D].double()
    want, size = R.attention(qd, k, ks, v, vs, kind, S.starts, S.total, S.table, S.P, H, attend.scale, window)
    o = got.cpu().double()[:S.tokens]
    assert bool(o.isfinite().all())
    # the largest sum |q k| over the keys of a head, as a bound for every row
    unit = 2.0**-24 * D + (2.0**-11 if dtype == torch.float32 else 0.0)
    kmax = (R.decode(k, kind).abs() * ks.double()[:, :, None, None]).amax((0, 2))  # [K, D]
    d = torch.zeros_like(qd)
    for h in range(H):
        at = slice(h * D, (h + 1) * D)
        d[:, at] = (abs(attend.scale) * (qd[:, at].abs() * kmax[h // G]).sum(1, keepdim=True) * unit)
    bound = (want.abs() * 2.0**-8 + size * (2.0**-10 + 2 * d))[:S.tokens] + 1e-30
    bound += (size.reshape(S.rows, H, D).amax(2, keepdim=True) * 2.0**-31 * max(S.total)).expand(-1, -1, D).reshape(S.rows, -1)[:S.tokens]
    far = (o - want[:S.tokens]).abs() / bound
    assert float(far.max()) <= 1.0, f"{float(far.max()):.2f} times the bound"


@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
def test_attention_of_single_tokens(lx, kind, D, P):
    S = R.Sequences([1] * 9 + [0], [1, 2, 15, 16, 17, P, P + 1, 3 * P - 1, 700, 40], P, seed=P, rows_behind=3)
    check_attention(lx, S, 2, 4, D, kind, seed=D)


@pytest.mark.parametrize("G", [1, 3, 7, 8, 9, 16, 24, 33, 64])
def test_attention_of_every_group(lx, G):
    S = R.Sequences([1, 1, 2], [300, 33, 130], 32, seed=G)
    check_attention(lx, S, 1, G, 128, "fp8", seed=G)
    check_attention(lx, S, 2, G, 64, "int8", seed=G, dtype=torch.float32)


@pytest.mark.parametrize("new,total", [([2, 4, 8], [2, 200, 1000]), ([5, 1, 0, 31], [5, 500, 64, 333]), ([130, 1, 64], [130, 300, 400]), ([257], [900]),
                                       ([1, 128, 129, 2], [1500, 128, 129, 700]), ([300, 40], [300, 41])])
@pytest.mark.parametrize("kind,D,G,window", [("fp8", 128, 4, 0), ("int8", 64, 7, 0), ("fp8", 64, 1, 100), ("int8", 128, 2, 17), ("fp8", 256, 3, 0), ("int8", 256, 1, 1)])
def test_attention_of_many_tokens(lx, new, total, kind, D, G, window):
    S = R.Sequences(new, total, 32, seed=len(new), rows_behind=1)
    check_attention(lx, S, 2, G, D, kind, window=window, seed=D + G)


@pytest.mark.parametrize("new,total", [([1, 1], [5000, 4097]), ([200], [6000]), ([3], [9001])])
@pytest.mark.parametrize("window", [0, 1, 64, 1000, 10**6])
def test_attention_over_long_caches(lx, new, total, window):
    S = R.Sequences(new, total, 64, seed=1)
    check_attention(lx, S, 1, 4, 128, "fp8", window=window, spread=4.0)


@pytest.mark.parametrize("new,total,D,K,G", [([257], [900], 64, 2, 7), ([300], [1500], 128, 1, 33), ([100, 130], [700, 800], 256, 2, 3), ([1, 1, 1], [900, 40, 3000], 128, 2, 4)])
def test_attention_gives_the_same_bits_in_many_calls(lx, new, total, D, K, G):
    """A copy that writes over what is still read, or a role that runs ahead of another, shows in one call of some hundred."""
    S = R.Sequences(new, total, 32, seed=1)
    cache, _ = make_cache(lx, S, K, D, "int8", 3)
    q, attend, batch = normal((S.rows, K * G * D), 5, dtype=torch.bfloat16).cuda(), host.Attention(cache, K * G), put(S)
    first = attend(batch, q)
    outs = [attend(batch, q) for _ in range(600)]
    util.check_status(lx)
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("max_new", [0, 1, 8, 10**6])
def test_attention_of_more_or_fewer_tokens_than_the_hint(lx, max_new):
    S = R.Sequences([150, 1, 9], [400, 100, 9], 16, seed=4)
    check_attention(lx, S, 2, 2, 64, "fp8", max_new=max_new)


@pytest.mark.parametrize("n", [1, 3, 200])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_attention_does_not_read_what_no_query_sees(lx, kind, n):
    """Slots past a sequence's end and before its window, pages of nobody and their scales hold codes and numbers that are not finite."""
    K, G, D, P, window = 2, 2, 128, 32, 50
    S = R.Sequences([n, n], [n + 71, n + 300], P, seed=6)
    k, ks = R.stored(S.pages, K, P, D, kind, 40)
    v, vs = R.stored(S.pages, K, P, D, kind, 41)
    wild = []
    for c, x in ((k, ks), (v, vs)):
        c, x = c.clone(), x.clone()
        seen = torch.zeros((S.pages, P), dtype=torch.bool)
        for s, (m, t) in enumerate(zip(S.new, S.total)):
            for slot in range(max(0, t - m - window + 1), t):
                seen[S.table[s][slot // P], slot % P] = True
        c[~seen[:, None].expand(-1, K, -1)] = 0x7F if kind == "fp8" else 0x80
        x[~seen.any(1)] = math.nan
        wild += [c, x]
    cache = host.KvCache(lx, WTYPE[kind], wild[0].cuda(), wild[2].cuda(), wild[1].cuda(), wild[3].cuda())
    # and the table entries before the window name no page
    for s, (m, t) in enumerate(zip(S.new, S.total)):
        S.matrix[s, :max(0, t - m - window + 1) // P] = -1
    check_attention(lx, S, K, G, D, kind, window=window, cache=(cache, (k, ks, v, vs)))


@pytest.mark.parametrize("n", [1, 40, 300])
def test_attention_rows_that_see_nothing_are_zero(lx, n):
    S = R.Sequences([n, 1], [n, 20], 16, seed=7)
    cache, parts = make_cache(lx, S, 1, 64, "fp8", 50)
    q = normal((S.rows, 4 * 64), 51, dtype=torch.bfloat16)
    attend = host.Attention(cache, 4)
    for length in (0, n // 2):
        out = attend(put(S, lengths=[length, 20]), q.cuda()).cpu()
        util.check_status(lx)
        assert bool((out[:n - length] == 0).all())
        want, _ = R.attention(q.double(), *parts, "fp8", S.starts, [length, 20], S.table, 16, 4, attend.scale, 0)
        assert float((out.double() - want).abs().max()) < 0.05 * float(want.abs().max())


@pytest.mark.parametrize("n", [1, 200])
def test_attention_over_a_page_outside_the_cache(lx, n):
    """The rows that see such a page are not-a-number and it is reported; the other sequences' rows are right."""
    S = R.Sequences([n, n], [n + 100, n + 40], 32, seed=8)
    cache, parts = make_cache(lx, S, 2, 128, "int8", 60)
    q = normal((S.rows, 4 * 128), 61, dtype=torch.bfloat16)
    attend = host.Attention(cache, 4)
    right = attend(put(S), q.cuda()).cpu()
    for page in (-1, S.pages, 2**31 - 1):
        S.matrix[0, 1] = page
        out = attend(put(S), q.cuda()).cpu()
        torch.cuda.synchronize()
        assert lx.lx_b200_last_error() == 9
        assert bool(out[:n].isnan().all())
        assert torch.equal(out[n:], right[n:])
    # and a table too short for the lengths, sequences of impossible rows
    batch = host.KvBatch(torch.tensor(S.starts, dtype=torch.int32).cuda(), torch.tensor(S.total, dtype=torch.int32).cuda(), S.matrix[:, :1].contiguous().cuda(),
                         tokens=S.rows, max_new=n)
    out = attend(batch, q.cuda()).cpu()
    torch.cuda.synchronize()
    assert lx.lx_b200_last_error() == 9 and bool(out.isnan().all())


def test_attention_reads_nan_where_a_scale_is(lx):
    """A page whose scale is not-a-number for one head: that head's rows that see it, and no others."""
    S = R.Sequences([1, 40], [90, 80], 32, seed=9)
    cache, parts = make_cache(lx, S, 2, 64, "fp8", 70)
    q = normal((S.rows, 4 * 64), 71, dtype=torch.bfloat16)
    attend = host.Attention(cache, 4)
    right = attend(put(S), q.cuda()).cpu()
    for scales in (cache.k_scale, cache.v_scale):
        page = S.table[1][2]  # slots 64 .. 79 of the second sequence
        was = scales[page, 1].clone()
        scales[page, 1] = math.nan
        out = attend(put(S), q.cuda()).cpu()
        scales[page, 1] = was
        util.check_status(lx)
        nan = out.isnan()
        want = torch.zeros_like(nan)
        want[1 + 24:, 2 * 64:] = True
        assert torch.equal(nan, want) and torch.equal(out[~nan], right[~nan])


def test_attention_where_scales_are_far_apart(lx):
    """Values of one page 2^60 times those of another, keys too: weights and sums hold their digits."""
    S = R.Sequences([1, 1, 70], [200, 130, 130], 16, seed=10)
    cache, (k, ks, v, vs) = make_cache(lx, S, 1, 128, "fp8", 80)
    vs[S.table[0][3]] *= 2.0**60
    vs[S.table[1][0]] *= 2.0**-60
    vs[S.table[2][1]] *= 2.0**-100 / float(vs[S.table[2][1]].max())
    ks[S.table[0][2]] *= 2.0**-30
    cache.v_scale.copy_(vs), cache.k_scale.copy_(ks)
    check_attention(lx, S, 1, 4, 128, "fp8", cache=(cache, (k, ks, v, vs)))


def test_attention_with_offsets_past_32_bits(lx):
    """Keys and values in one pool whose pages are 80 MB apart: the last ones begin past 2^32 bytes."""
    K, D, P, kind = 2, 64, 16, "fp8"
    S = R.Sequences([2, 1], [500, 350], P, seed=11)
    assert S.pages > 54
    k, ks = R.stored(S.pages, K, P, D, kind, 90)
    v, vs = R.stored(S.pages, K, P, D, kind, 91)
    stride, page = 80 * 2**20, K * P * D
    pool = torch.empty(S.pages * stride, dtype=torch.uint8, device="cuda")
    views = [pool.as_strided((S.pages, K, P, D), (stride, P * D, D, 1), off) for off in (0, page)]
    views[0].copy_(k), views[1].copy_(v)
    cache = host.KvCache(lx, WTYPE[kind], *views, ks.cuda(), vs.cuda())
    check_attention(lx, S, K, 2, D, kind, cache=(cache, (k, ks, v, vs)))
    x = normal((S.rows, K * D), 92)
    cache.append(put(S), x.cuda(), x.cuda())
    util.check_status(lx)
    want, scale = R.append(v, vs, kind, x.double().reshape(S.rows, K, D), S.starts, S.total, S.table, P)
    assert torch.equal(views[1].cpu(), want) and torch.equal(cache.v_scale.cpu(), scale)


@pytest.mark.parametrize("n", [1, 60])
@pytest.mark.parametrize("scale", [-0.11, 0.0, 1.5])
def test_attention_with_any_scale(lx, n, scale):
    S = R.Sequences([n, 1], [n + 150, 77], 16, seed=12)
    check_attention(lx, S, 2, 2, 128, "int8", scale=scale, spread=0.5)
    check_attention(lx, S, 1, 4, 64, "fp8", scale=scale, spread=0.5, window=30, dtype=torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_that_begin_anywhere(lx, dtype):
    """Odd offsets and strides of queries, keys, values and results: the same values as rows on 16 bytes."""
    K, G, D, P = 2, 3, 64, 16
    W, KV = K * G * D, K * D
    for n in (1, 90):
        S = R.Sequences([n, 2], [n + 50, 40], P, seed=13)
        rows = normal((S.rows, W + 2 * KV), 14, dtype=dtype).cuda()
        odd = torch.full((S.rows, W + 2 * KV + 5), 3.0, dtype=dtype, device="cuda")[:, 3:-2]
        odd.copy_(rows)
        caches = [make_cache(lx, S, K, D, "fp8", 15)[0] for _ in range(2)]
        one = host.Rotary.of(32, device="cuda")
        batch, outs = put(S), []
        for cache, x in zip(caches, (rows, odd)):
            q_out = torch.zeros((S.rows, W + 7), dtype=dtype, device="cuda")[:, 1:W + 1] if x is odd else torch.zeros((S.rows, W), dtype=dtype, device="cuda")
            q = cache.append(batch, x[:, W:W + KV], x[:, W + KV:], q=x[:, :W], rotary=one, q_out=q_out)
            out = torch.zeros((S.rows, W + 9), dtype=torch.bfloat16, device="cuda")[:, 5:W + 5] if x is odd else torch.zeros((S.rows, W), dtype=torch.bfloat16, device="cuda")
            outs.append((q.clone(), host.Attention(cache, K * G)(batch, q, out=out).clone(), cache.k.clone(), cache.v.clone(), cache.k_scale.clone(), cache.v_scale.clone()))
        util.check_status(lx)
        assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_many_sequences(lx):
    """More sequences than a CTA has threads, some of them with many new tokens, some with none."""
    g = torch.Generator().manual_seed(16)
    total = torch.randint(1, 200, (333,), generator=g).tolist()
    new = [0 if i % 7 == 3 else min(t, 40) if i % 50 == 0 else 1 for i, t in enumerate(total)]
    S = R.Sequences(new, total, 16, seed=17, rows_behind=2)
    check_attention(lx, S, 2, 4, 64, "fp8", max_new=1)
    check_attention(lx, S, 2, 4, 64, "int8")
    K, D = 2, 64
    x = normal((S.rows, K * D), 18)
    for hint in (1, 40):
        cache, (k0, ks0, v0, vs0) = make_cache(lx, S, K, D, "int8", 19)
        cache.append(put(S, max_new=hint), x.cuda(), x.cuda())
        util.check_status(lx)
        v, vs = R.append(v0, vs0, "int8", x.double().reshape(S.rows, K, D), S.starts, S.total, S.table, 16)
        assert torch.equal(cache.v.cpu(), v) and torch.equal(cache.v_scale.cpu(), vs)


# ---- norms -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,C", [(1, 4096), (3, 8), (2, 1), (5, 1000), (33, 2048), (2, 8192), (3, 8200), (2, 16384), (2, 16392), (7, 4097), (300, 4096), (310, 5000), (300, 16384)])
@pytest.mark.parametrize("y,h,w,gate,sigmoid,post,x", [
    ("f32", "f32", "bf16", None, False, True, "bf16"), ("bf16", "bf16", "f32", "channel", False, True, "f32"), ("f32", "bf16", "bf16", "token", True, True, "bf16"),
    ("bf16", "f32", "f32", "token", False, False, "bf16"), (None, "f32", "bf16", None, False, False, "f32")])
def test_norm(lx, T, C, y, h, w, gate, sigmoid, post, x):
    of = {"f32": torch.float32, "bf16": torch.bfloat16}
    yt = None if y is None else normal((T, C + 24), 1, 2.0, of[y])
    ht = normal((T, C + 8), 2, 3.0, of[h])
    gt = None if gate is None else normal((C,) if gate == "channel" else (T, C), 3, 1.0, torch.bfloat16)
    pre, pt = 1 + normal((C,), 4, 0.2, of[w]), 1 + normal((C,), 5, 0.2, of[w])
    layer = host.NormResidual(lx, C, pre=pre.cuda(), post=pt.cuda() if post else None, residual_scale=0.75, block_scale=1.25, gate_sigmoid=sigmoid, eps=1e-5)
    args = [None if yt is None else yt.cuda()[:, :C], ht.cuda()[:, :C]]
    xt = torch.empty((T, C), dtype=of[x], device="cuda")
    h2, x2 = layer(*args, gate=None if gt is None else gt.cuda(), x=xt)
    assert x2 is xt and h2.dtype == of[h]
    want_h, want_x, a, b = R.norm(None if yt is None else yt[:, :C].double(), ht[:, :C].double(), None if gt is None else gt.double(), pt.double() if post else None,
                                  pre.double(), 0.75, 1.25, sigmoid, 1e-5)
    near = 2.0**-19
    assert bool(((h2.cpu().double() - want_h).abs() <= (a + b) * near + want_h.abs() * (2.0**-8 if h == "bf16" else 0)).all())
    # x = h' times a factor that is 2^-19 off at most, h' off by (a + b) 2^-19
    factor = want_x.abs() / want_h.abs().clamp(min=1e-30)
    assert bool(((x2.cpu().double() - want_x).abs() <= factor * (a + b) * near + want_x.abs() * (near + (2.0**-8 if x == "bf16" else 2.0**-24))).all())
    # in place, and a row alone has the bits that it has among others
    buf = args[1].clone()
    h3, x3 = layer(*args[:1], buf, gate=None if gt is None else gt.cuda(), h_out=buf, x=torch.empty_like(xt))
    assert h3 is buf and torch.equal(h3, h2) and torch.equal(x3, x2)
    one = layer(None if yt is None else args[0][T - 1:], args[1][T - 1:], gate=None if gt is None else gt.cuda() if gate == "channel" else gt.cuda()[T - 1:],
                x=torch.empty_like(xt[:1]))
    assert torch.equal(one[0], h2[T - 1:]) and torch.equal(one[1], x2[T - 1:])
    util.check_status(lx)


def test_norm_without_a_next_norm_and_of_rows_of_zeros(lx):
    h, y = normal((4, 512), 1).cuda(), torch.zeros((4, 512), device="cuda")
    layer = host.NormResidual(lx, 512, post=torch.ones(512, device="cuda"))
    h2, x = layer(y, h)
    assert x is None and torch.equal(h2, h)
    layer = host.NormResidual(lx, 512, pre=torch.ones(512, device="cuda"), post=torch.ones(512, device="cuda"))
    h2, x = layer(y, torch.zeros_like(h))
    assert bool((h2 == 0).all()) and bool((x == 0).all())
    y[1, 7] = math.nan
    h2, x = layer(y, h)
    assert bool(x[1].isnan().all()) and bool(x[[0, 2, 3]].isfinite().all())


# ---- together ----------------------------------------------------------------------------------------------------------------
def make_block(lx, kind, D, K, G, width, P, pages, wtype=abi.W_BF16):
    H = K * G
    wq = (normal(((H + 2 * K) * D, width), 1, width**-0.5)).to(torch.bfloat16)
    wo = (normal((width, H * D), 2, (H * D)**-0.5)).to(torch.bfloat16)
    cache = host.KvCache.empty(lx, WTYPE[kind], pages, K, D, P)
    norm = host.NormResidual(lx, width, pre=1 + normal((width,), 3, 0.1).cuda(), post=1 + normal((width,), 4, 0.1).cuda(), residual_scale=0.9)
    block = host.AttentionBlock(host.Linear(lx, host.store_weight(lx, wq.cuda(), wtype), (H + 2 * K) * D, width),
                                host.Linear(lx, host.store_weight(lx, wo.cuda(), wtype), width, H * D), cache, H, norm, rotary=host.Rotary.of(D, device="cuda"))
    return block, wq.double(), wo.double()


@pytest.mark.parametrize("kind,D,G,P", [("fp8", 64, 4, 16), ("int8", 128, 2, 32)])
def test_a_layer_decodes_what_it_would_have_computed_at_once(lx, kind, D, G, P):
    """A prompt in one call, then tokens one at a time, against the layer's formula in 64 bits over unrounded keys and values. What the
    cache's codes cost is what the tolerance counts: 2^-4 of a value in E4M3, half a step of 1/64 of a page's largest value in INT8,
    averaged by the softmax; outputs are compared by their norms, at a tenth of the block's output."""
    K, width, prompt, steps = 2, 512, 40, 9
    block, wq, wo = make_block(lx, kind, D, K, G, width, P, 8)
    H, T = K * G, prompt + steps
    x, h = normal((T, width), 5).to(torch.bfloat16), normal((T, width), 6)
    table = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32).cuda()
    lengths = torch.tensor([prompt], dtype=torch.int32).cuda()
    outs = [block(x[:prompt].cuda(), h[:prompt].cuda(), host.KvBatch(torch.tensor([0, prompt], dtype=torch.int32).cuda(), lengths, table, prompt, prompt))]
    one = host.KvBatch(torch.tensor([0, 1], dtype=torch.int32).cuda(), lengths, table, 1, 1)
    for t in range(prompt, T):
        lengths.fill_(t + 1)
        outs.append(block(x[t:t + 1].cuda(), h[t:t + 1].cuda(), one))
    util.check_status(lx)
    got_h, got_x = (torch.cat([o[i] for o in outs]).cpu().double() for i in (0, 1))
    rows = x.double() @ wq.T
    turned = R.rotate(rows[:, :(H + K) * D].reshape(T, H + K, D), torch.arange(T), block.rotary.frequencies.cpu(), False)
    v = rows[:, (H + K) * D:].reshape(T, K, D)
    o = torch.zeros(T, H, D, dtype=torch.float64)
    hidden = torch.ones(T, T).triu(1).bool()
    for i in range(H):
        s = (turned[:, i] @ turned[:, H + i // G].T * D**-0.5).masked_fill(hidden, -math.inf)
        o[:, i] = s.softmax(1) @ v[:, i // G]
    want_h, want_x, _, b = R.norm(o.reshape(T, -1) @ wo.T, h.double(), None, block.norm.post.cpu().double(), block.norm.pre.cpu().double(), 0.9, 1.0, False, 1e-6)
    assert float((got_h - want_h).norm()) <= 0.1 * float(b.norm())
    assert float((got_x - want_x).norm()) <= 0.1 * float(want_x.norm())


def test_a_captured_layer_follows_its_lengths(lx):
    """A decode step captured in a graph and replayed for token after token, on a stream of its own, while eager calls of another layer run
    beside it, gives what eager steps give."""
    K, G, D, P, width = 2, 4, 128, 16, 256
    results = []
    for captured in (False, True):
        block, _, _ = make_block(lx, "fp8", D, K, G, width, P, 40)
        beside, _, _ = make_block(lx, "int8", D, K, G, width, P, 40)
        S = 3
        table = torch.randperm(40, generator=torch.Generator().manual_seed(1))[:36].reshape(S, 12).to(torch.int32).cuda()
        starts, lengths = torch.arange(S + 1, dtype=torch.int32).cuda(), torch.zeros(S, dtype=torch.int32).cuda()
        batch = host.KvBatch(starts, lengths, table, S, 1)
        x, h = torch.empty((S, width), dtype=torch.bfloat16, device="cuda"), torch.empty((S, width), device="cuda")
        x.copy_(normal((S, width), 11)), h.copy_(normal((S, width), 12))
        for b in (block, beside):  # workspaces and modules, and slots that are written again
            lengths.fill_(1)
            b(x, h, batch)
        torch.cuda.synchronize()
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        if captured:
            with torch.cuda.graph(graph):
                step = block(x, h, batch)
        lengths.copy_(torch.tensor([0, 50, 17]))
        got = []
        with torch.cuda.stream(stream):
            stream.wait_stream(torch.cuda.default_stream())
            for t in range(40):
                x.copy_(normal((S, width), 200 + t).cuda()), h.copy_(normal((S, width), 300 + t).cuda())
                lengths.add_(1)
                torch.cuda.default_stream().wait_stream(stream)
                with torch.cuda.stream(torch.cuda.default_stream()):
                    beside(x, h, batch)
                if captured:
                    graph.replay()
                    out = step
                else:
                    out = block(x, h, batch)
                stream.wait_stream(torch.cuda.default_stream())
                got.append(torch.cat([out[0], out[1].float()], 1).clone())
        torch.cuda.synchronize()
        results.append(torch.cat(got))
        util.check_status(lx)
        del graph
    assert bool(results[0].isfinite().all()) and torch.equal(results[0], results[1])
