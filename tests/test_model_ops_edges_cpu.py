# SPDX-License-Identifier: Apache-2.0
"""The model operators where they can go wrong, as far as that shows without a GPU."""

from vkccl_b200._lib import lib


def test_attention_status_with_nothing_launched():
    assert lib().vcclKv4AttentionStatus() == 0
