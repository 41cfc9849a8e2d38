"""Sizes that no launch of the token operators can hold are refused before any device work, like the other refusals of
test_tokens.py."""
import ctypes

import pytest

import test_tokens as T
import vknn_amd as V

R = ctypes.byref


@pytest.mark.parametrize("change", [dict(q_heads=1 << 24, kv_heads=1, total_q=1), dict(q_heads=1 << 25, kv_heads=1, total_q=1), dict(q_heads=1 << 24, kv_heads=1 << 24, total_q=100)])
def test_attention_refuses_more_heads_than_a_launch(change):
    d = V.AttentionDesc(**{**T.AT, **change})
    T.refused(V.vkhip().vkhip_attention_packed(R(d), T.A, T.A, T.A, T.A, T.A, T.A, T.A, None), "attention_packed")
    assert V.vkhip().vkhip_attention_workspace_bytes(R(d)) == 0
