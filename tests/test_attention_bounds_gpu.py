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
