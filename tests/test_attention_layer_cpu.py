"""What the attention layer's operators refuse, at the C ABI and at the host's classes, without a GPU: no call here reaches a launch.
And the plain implementations that the GPU tests compare with, checked against simple cases."""

import ctypes

import pytest
import torch

from dromos_b200 import abi, host
from tests import kv_reference as R


@pytest.fixture(scope="module")
def lib():
    return abi.Library(abi.default_library_path())


def cache(**kw):
    a = dict(type=abi.W_FP8, kv_heads=2, head_dim=64, page_tokens=16, pages=4, page_stride=2048, k=4096, v=8192, k_scale=64, v_scale=128)
    assert set(kw) <= set(a)
    a.update(kw)
    return abi.KvCacheStruct(*a.values())


def batch(**kw):
    a = dict(sequences=1, tokens=0, max_new=1, ld_pages=1, starts=64, lengths=64, pages=64)
    assert set(kw) <= set(a)
    a.update(kw)
    return abi.KvBatchStruct(*a.values())


def address(x):
    return None if x is None else ctypes.addressof(x)


def append(lib, c, b, **kw):
    a = dict(k=64, ld_k=128, v=64, ld_v=128, dtype=0, q=64, q_dtype=0, ld_q=256, q_heads=4, q_out=64, q_out_dtype=1, ld_q_out=256, positions=None, frequencies=64,
             rotary_dim=64, interleaved=0, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lx_b200_kv_append(address(c), address(b), *a.values())


def attend(lib, c, b, **kw):
    a = dict(q=64, q_dtype=1, ld_q=256, q_heads=4, scale=1.0, window=0, out=64, ld_out=256, workspace=4096, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lx_b200_attention(address(c), address(b), *a.values())


def norm(lib, **kw):
    a = dict(y=64, y_dtype=0, ld_y=32, h=64, h_dtype=0, ld_h=32, gate=None, gate_dtype=0, ld_gate=0, gate_sigmoid=0, post=64, pre=64, weight_dtype=0, residual_scale=1.0,
             block_scale=1.0, eps=1e-6, h_out=64, ld_h_out=32, x=64, x_dtype=1, ld_x=32, T=0, C=32, stream=None)
    assert set(kw) <= set(a)
    a.update(kw)
    return lib.lx_b200_norm_residual(*a.values())


BAD_CACHES = [dict(kv_heads=0), dict(pages=0), dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(page_stride=2032), dict(page_stride=2056),
              dict(k=4104), dict(v=8200), dict(k_scale=66)]
UNSUPPORTED_CACHES = [dict(type=abi.W_BF16), dict(type=abi.W_NVFP4), dict(head_dim=80), dict(head_dim=0), dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256),
                      dict(kv_heads=2000, page_stride=10**7), dict(pages=2**32)]
BAD_BATCHES = [dict(sequences=-1), dict(tokens=-1), dict(max_new=-1), dict(ld_pages=-1), dict(starts=None), dict(lengths=None), dict(pages=None)]


@pytest.mark.parametrize("call", [append, attend])
def test_caches_and_batches_that_are_refused(lib, call):
    assert call(lib, cache(), batch()) == 0  # no rows: nothing to launch
    assert call(lib, cache(), batch(sequences=0, starts=None, lengths=None, pages=None, tokens=9)) == 0
    assert call(lib, None, batch()) == abi.ERR_INVALID and call(lib, cache(), None) == abi.ERR_INVALID
    for kw in BAD_CACHES:
        assert call(lib, cache(**kw), batch(tokens=4)) == abi.ERR_INVALID, kw
    for kw in UNSUPPORTED_CACHES:
        assert call(lib, cache(**kw), batch(tokens=4)) == abi.ERR_NOT_SUPPORTED, kw
    for kw in BAD_BATCHES:
        assert call(lib, cache(), batch(**kw)) == abi.ERR_INVALID, kw


def test_appends_that_are_refused(lib):
    for kw in (dict(k=None), dict(v=None), dict(ld_k=127), dict(ld_v=127), dict(dtype=2), dict(q_dtype=-1), dict(q_out_dtype=9), dict(q_heads=0), dict(q_heads=3),
               dict(q_out=None), dict(ld_q=255), dict(ld_q_out=255), dict(frequencies=None), dict(rotary_dim=-8), dict(rotary_dim=72)):
        assert append(lib, cache(), batch(tokens=4), **kw) == abi.ERR_INVALID, kw
    assert append(lib, cache(), batch(tokens=4), rotary_dim=20) == abi.ERR_NOT_SUPPORTED


def test_attentions_that_are_refused(lib):
    for kw in (dict(q=None), dict(out=None), dict(ld_q=255), dict(ld_out=255), dict(q_dtype=2), dict(q_heads=0), dict(q_heads=5), dict(window=-1), dict(workspace=None), dict(workspace=4096 + 128)):
        assert attend(lib, cache(), batch(tokens=4), **kw) == abi.ERR_INVALID, kw
    assert lib.lx_b200_attention_workspace_bytes(address(cache()), address(batch()), 4) >= 0
    for args in ((None, batch(), 4), (cache(), None, 4), (cache(), batch(), 5), (cache(), batch(), 0), (cache(), batch(max_new=-1), 4), (cache(head_dim=80), batch(), 4)):
        assert lib.lx_b200_attention_workspace_bytes(address(args[0]), address(args[1]), args[2]) == -1


def test_norms_that_are_refused(lib):
    assert norm(lib) == 0
    for kw in (dict(T=-1), dict(C=0), dict(y_dtype=2), dict(h_dtype=-1), dict(gate_dtype=5), dict(weight_dtype=2), dict(x_dtype=7)):
        assert norm(lib, **kw) == abi.ERR_INVALID, kw
    for kw in (dict(h=None), dict(x=None), dict(h_out=None, pre=None), dict(ld_y=31), dict(ld_h=31), dict(gate=64, ld_gate=31), dict(ld_h_out=31), dict(ld_x=31)):
        assert norm(lib, T=4, **kw) == abi.ERR_INVALID, kw


def test_the_host_refuses_buffers_that_do_not_fit(lib):
    codes, scale = torch.zeros((4, 2, 16, 64), dtype=torch.uint8), torch.ones((4, 2))
    ok = host.KvCache(lib, abi.W_FP8, codes, codes.clone(), scale, scale.clone())
    for args in ((codes[:, :, ::2], codes, scale, scale), (codes, codes[:3], scale, scale), (codes.float(), codes, scale, scale), (codes, codes, scale.double(), scale),
                 (codes, codes, scale, scale[:, :1])):
        with pytest.raises(ValueError):
            host.KvCache(lib, abi.W_FP8, *args)
    starts, lengths, pages = (torch.zeros(n, dtype=torch.int32) for n in ((3,), (2,), (2, 5)))
    b = host.KvBatch(starts, lengths, pages, 4, 2)
    for args in ((starts[:2], lengths, pages), (starts.long(), lengths, pages), (starts, lengths, pages[:1]), (starts, lengths, pages.T.contiguous().T), (starts, lengths[::2], pages)):
        with pytest.raises(ValueError):
            host.KvBatch(*args, 4, 2)
    with pytest.raises(ValueError):
        host.KvBatch(starts, lengths, pages, -1, 2)
    with pytest.raises(ValueError):
        host.Rotary(torch.ones(4))
    with pytest.raises(ValueError):
        host.Attention(ok, 5)
    with pytest.raises(ValueError):
        host.NormResidual(lib, 32, pre=torch.ones(31))
    with pytest.raises(TypeError):
        host.NormResidual(lib, 32, pre=torch.ones(32, dtype=torch.float16))
    rows = torch.zeros((4, 128))
    # buffers that are not on the current CUDA device are refused before anything is launched
    for call in (lambda: ok.append(b, rows, rows), lambda: host.Attention(ok, 2)(b, rows), lambda: host.NormResidual(lib, 128)(rows, rows)):
        with pytest.raises(ValueError):
            call()


def test_row_strides():
    x, cpu = torch.zeros((4, 24)), torch.device("cpu")
    assert host._rows(x[:, :8], 4, 8, "x", cpu) == 24 and host._rows(x[:1, :8], 1, 8, "x", cpu) == 24 and host._rows(x[:, :24], 4, 24, "x", cpu) == 24
    assert host._rows(x[:1, :1], 1, 1, "x", cpu) == 24 and host._rows(x[:, ::24], 4, 1, "x", cpu) == 24
    for bad in (x[:, ::2], x[:2], x[:, :7], x[:, None]):
        with pytest.raises(ValueError):
            host._rows(bad, 4, 12, "x", cpu)
    with pytest.raises(ValueError):
        host._rows(x, 4, 24, "x", torch.device("cuda", 0))


# ---- the plain implementations -------------------------------------------------------------------------------------------------
def test_plain_codes_round_to_nearest_even():
    x = torch.tensor([0.0, 1.0, 1.0624, 1.0625, 1.0626, 1.1875, 447.0, 448.0, 500.0, -2.0**-10, -2.0**-10 * 1.01, 1.0625 + 2.0**-40, 1.1875 - 2.0**-40], dtype=torch.float64)
    want = [0, 1, 1, 1, 1.125, 1.25, 448, 448, 448, 0, -2.0**-9, 1.125, 1.125]
    assert R.decode(R.encode(x, "fp8"), "fp8").tolist() == want
    assert R.decode(R.encode(torch.tensor([0.5, 1.5, -2.5, 126.6, 300.0], dtype=torch.float64), "int8"), "int8").tolist() == [0, 2, -2, 127, 127]
    for kind, top in R.TOP.items():
        assert R.power_of_two(top, kind) == 1.0 and R.power_of_two(top * 1.0001, kind) == 2.0 and R.power_of_two(top / 2, kind) == 0.5 and R.power_of_two(0.0, kind) == 2.0**-100


def test_plain_append_and_attention_agree_with_a_dense_softmax():
    K, D, P, n, t = 2, 64, 16, 5, 21
    S = R.Sequences([n], [t], P, seed=1)
    g = torch.Generator().manual_seed(2)
    x = torch.randn((t, K, D), generator=g, dtype=torch.float64)
    k, ks = R.stored(S.pages, K, P, D, "int8", 3)
    k, ks = R.append(k, ks, "int8", x, [0, t], [t], S.table, P)
    held = (R.decode(k[S.table[0]], "int8") * ks[S.table[0]].double()[:, :, None, None]).transpose(0, 1).reshape(K, -1, D)[:, :t]
    assert float((held.transpose(0, 1) - x).abs().max()) <= float(ks.max()) / 2
    q = torch.randn((n, 4 * D), generator=g, dtype=torch.float64)
    out, size = R.attention(q, k, ks, k, ks, "int8", [0, n], [t], S.table, P, 4, 0.125, 0)
    hidden = torch.arange(t)[None] > torch.arange(t - n, t)[:, None]
    want = torch.stack([((q[:, h * D:(h + 1) * D] @ held[h // 2].T) * 0.125).masked_fill(hidden, float("-inf")).softmax(1) @ held[h // 2] for h in range(4)], 1).reshape(n, -1)
    assert torch.allclose(out, want) and bool((size >= out.abs() - 1e-12).all())


def test_plain_rotation_turns_pairs():
    x = torch.tensor([[[1.0, 2.0, 3.0, 4.0, 5.0, 6.0]]], dtype=torch.float64)
    f = torch.tensor([0.5, 0.25], dtype=torch.float64)
    c, s = torch.cos(2 * f), torch.sin(2 * f)
    halves = R.rotate(x, torch.tensor([2]), f, False)[0, 0]
    assert torch.allclose(halves[:4], torch.stack([1 * c[0] - 3 * s[0], 2 * c[1] - 4 * s[1], 3 * c[0] + 1 * s[0], 4 * c[1] + 2 * s[1]])) and halves[4:].tolist() == [5, 6]
    pairs = R.rotate(x, torch.tensor([2]), f, True)[0, 0]
    assert torch.allclose(pairs[:4], torch.stack([1 * c[0] - 2 * s[0], 2 * c[0] + 1 * s[0], 3 * c[1] - 4 * s[1], 4 * c[1] + 3 * s[1]]))
