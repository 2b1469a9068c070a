"""A norm row's bits whatever the other rows: few rows and many go through different kernels."""

import itertools

import pytest
import torch

from dromos_b200 import host
from tests import util
from tests.test_attention_layer_gpu import normal

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("C", [8, 1000, 4096, 8192, 16384, 1001])
def test_rows_alone_and_among_many_have_the_same_bits(lx, C):
    T, few = 2 * torch.cuda.get_device_properties(0).multi_processor_count + 4, slice(5, 8)
    y, h, rows, channel = normal((T, C), 1, 2.0).cuda(), normal((T, C), 2, 3.0).cuda(), normal((T, C), 3).cuda(), normal((C,), 4).cuda()
    pre, post = 1 + normal((C,), 5, 0.2).cuda(), 1 + normal((C,), 6, 0.2).cuda()
    for y_type, h_type, normed, gate, sigmoid in itertools.product((torch.float32, torch.bfloat16, None), (torch.float32, torch.bfloat16), (True, False),
                                                                    (None, "channel", "rows"), (True, False)):
        layer = host.NormResidual(lx, C, pre=pre, post=post if normed else None, residual_scale=0.7, block_scale=1.3, gate_sigmoid=sigmoid)
        yt, ht = None if y_type is None else y.to(y_type), h.to(h_type)
        g = {None: None, "channel": channel, "rows": rows}[gate]
        many = layer(yt, ht, gate=g, x=torch.empty_like(h))
        alone = layer(None if yt is None else yt[few], ht[few], gate=g[few] if gate == "rows" else g, x=torch.empty_like(h[few]))
        for a, b in zip(many, alone):
            assert torch.equal(a[few].view(torch.int16), b.view(torch.int16)), (y_type, h_type, normed, gate, sigmoid)
    util.check_status(lx)
