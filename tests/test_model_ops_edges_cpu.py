# SPDX-License-Identifier: Apache-2.0
"""The model operators where they can go wrong, as far as that shows without a GPU."""

import pytest
import torch

from vkccl_b200._lib import lib
from vkccl_b200.ops import _args
from vkccl_b200.ops.rope import qk_norm_rope


def test_attention_status_with_nothing_launched():
    assert lib().vcclKv4AttentionStatus() == 0


@pytest.mark.parametrize("which", range(4))
def test_norm_rope_refuses_to_lose_a_gradient(which):
    x = [torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.zeros(4, 1, 64, dtype=torch.bfloat16),
         torch.ones(64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)]
    x[which].requires_grad_()
    pos, freq = torch.zeros(4, dtype=torch.int32), torch.zeros(32)
    with pytest.raises(ValueError, match="history"):
        qk_norm_rope(x[0], x[1], pos, freq, q_weight=x[2], k_weight=x[3])
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # the next check: these are CPU tensors
        qk_norm_rope(x[0], x[1], pos, freq, q_weight=x[2], k_weight=x[3])


@pytest.mark.parametrize("tokens", [2**31 - 1, 2**30 + 1])
def test_more_rows_than_an_int_holds_in_blocks_are_refused(tokens):
    """Row numbers rounded up to whole blocks would pass 2^31: every entry returns vcclInvalidArgument before it launches."""
    from test_model_ops_cpu import BF16, INVALID, P, cache_c, heads, plan, rope_c

    h, one = lib(), heads(n=1, tok=128)
    c = cache_c(n=1)
    assert plan(tokens=tokens) == INVALID
    assert h.vcclQkNormRope(one, one, rope_c(), one, one, tokens, 128, BF16, None) == INVALID
    assert h.vcclQkNormRopeBackward(one, one, one, one, rope_c(), one, one, None, None, None, tokens, 128, BF16, None) == INVALID
    assert h.vcclKv4Append(c, one, one, P, None, None, None, tokens, BF16, None) == INVALID
    assert h.vcclKv4Read(c, P, one, one, tokens, BF16, None) == INVALID
    assert h.vcclKv4Attention(one, c, P, 2, P, P, 2, tokens, 0.1, one, None, 1, P, BF16, None) == INVALID
    with pytest.raises(ValueError, match="2\\^30"):
        _args.heads(torch.zeros(1, 1, 64, dtype=torch.bfloat16).expand(tokens, 1, 64), "x", torch.bfloat16, -1, tokens, 64)
