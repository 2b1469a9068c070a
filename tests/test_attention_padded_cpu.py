"""What lx_b200_attention_padded refuses: what lx_b200_attention does; and what no batch can hold. No call here reaches a launch."""

import pytest

from dromos_b200 import abi
from tests.test_attention_layer_cpu import BAD_BATCHES, BAD_CACHES, UNSUPPORTED_CACHES, address, append, attend, batch, cache


class Padded:
    """The library as `attend` sees it, with the padded call in the place of the other."""

    def __init__(self):
        self.lx_b200_attention = abi.Library(abi.default_library_path()).lx_b200_attention_padded


@pytest.fixture(scope="module")
def lib():
    return Padded()


def test_padded_attentions_that_are_refused(lib):
    assert attend(lib, cache(), batch()) == 0 and attend(lib, cache(), batch(sequences=0, starts=None, lengths=None, pages=None)) == 0  # no rows
    assert attend(lib, None, batch()) == abi.ERR_INVALID and attend(lib, cache(), None) == abi.ERR_INVALID
    for kws, answer in ((BAD_CACHES, abi.ERR_INVALID), (UNSUPPORTED_CACHES, abi.ERR_NOT_SUPPORTED)):
        for kw in kws:
            assert attend(lib, cache(**kw), batch(tokens=4)) == answer, kw
    for kw in BAD_BATCHES:
        assert attend(lib, cache(), batch(**kw)) == abi.ERR_INVALID, kw
    for b in (batch(tokens=4), batch(tokens=4, sequences=0, starts=None, lengths=None, pages=None)):
        for kw in (dict(q=None), dict(out=None), dict(ld_q=255), dict(ld_out=255), dict(q_dtype=2), dict(q_heads=0), dict(q_heads=5), dict(window=-1), dict(workspace=None),
                   dict(workspace=4096 + 128)):
            assert attend(lib, cache(), b, **kw) == abi.ERR_INVALID, kw


@pytest.mark.parametrize("sequences", [2**30 + 1, 2**31 - 128, 2**31 - 1])
def test_more_sequences_than_the_kernels_count(sequences):
    """Their loops over sequences count in steps of a CTA's threads, in 32 bits, and the order of work has a place for each."""
    lib, b = abi.Library(abi.default_library_path()), batch(tokens=4, sequences=sequences)
    assert attend(lib, cache(), b) == abi.ERR_NOT_SUPPORTED and attend(Padded(), cache(), b) == abi.ERR_NOT_SUPPORTED
    assert append(lib, cache(), b) == abi.ERR_NOT_SUPPORTED
    assert lib.lx_b200_attention_workspace_bytes(address(cache()), address(b), 4) == -1
