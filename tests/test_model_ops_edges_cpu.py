# SPDX-License-Identifier: Apache-2.0
"""The model operators where they can go wrong, as far as that shows without a GPU."""

import pytest
import torch

from vkccl_b200._lib import lib
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
