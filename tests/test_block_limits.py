"""The expert block's entries at the ends of their ranges, as far as no device call is needed."""
from __future__ import annotations

import pytest

import raggedroute_amd as rr

P = 4096  # a pointer that is never followed


@pytest.mark.parametrize("tokens", [1, 2048, 2 ** 20 + 1, 2 ** 30, 2 ** 30 + 5, 2 ** 31 - 2048, 2 ** 31 - 1])
@pytest.mark.parametrize("gate_tokens", [0, 1, 2047, 2 ** 30 - 1, 2 ** 30 + 1, 1500000000, 2 ** 31 - 1])
def test_norm_workspace_of_many_tokens(tokens, gate_tokens):
    """Three FP32 sums a column and part. A row of one value takes 64 threads and all parts
    together 131072: parts of ceil(tokens / 2048) tokens, gate rows cut into equal parts of at
    most that many or parts of whole gate rows."""
    def divide(a, by):
        return -(-a // by)

    args = rr.BlockNormBackwardArgs(h=P, block=P, gate=P if gate_tokens else None, gate_tokens=gate_tokens, dh=P, dx=P,
                                    tokens=tokens, hidden=1)
    most, group = divide(tokens, 2048), min(gate_tokens or tokens, tokens)
    if group >= most:
        cut = divide(group, divide(group, most))
        parts = divide(tokens, group) * divide(group, cut)
    else:
        parts = divide(tokens, most // group * group)
    assert rr.get_block_norm_backward_workspace_size(args) == parts * 3 * 4


@pytest.mark.parametrize("field", ["dpre_weight", "dpost_weight"])
def test_norm_sums_of_no_tokens_are_aligned(field):
    args = rr.BlockNormBackwardArgs(**{field: P + 1}, tokens=0, hidden=8)
    status = rr.block_norm_backward(args, rr.RuntimeContext(architecture=int(rr.DeviceArchitecture.kGfx950)))
    assert status.code == rr.StatusCode.kInvalidArgument and "aligned" in status.message
