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


# Outputs whose rows or heads lie on each other: threads would write the same memory in any order.
@pytest.mark.parametrize("change", [dict(o_row=0), dict(o_row=56), dict(o_head=0), dict(o_head=56), dict(o_row=128, o_head=128), dict(o_row=120, o_head=64), dict(o_row=64, o_head=64 + 56)])
def test_attention_refuses_output_rows_on_each_other(change):
    lib, d = V.vkhip(), V.AttentionDesc(**{**T.AT, **change})
    T.refused(lib.vkhip_attention_packed(R(d), T.A, T.A, T.A, T.A, T.A, T.A, T.A, None), "attention_packed")
    assert lib.vkhip_attention_workspace_bytes(R(d)) == 0


@pytest.mark.parametrize("change", [dict(k_row=0), dict(v_row=56), dict(k_head=0), dict(v_head=56), dict(k_row=64, k_head=64), dict(v_row=64, v_head=120)])
def test_kv_read_refuses_rows_on_each_other(change):
    rows = V.KvRows(**{**dict(dtype=0, total=4, k_row=128, k_head=64, v_row=128, v_head=64), **change})
    T.refused(V.vkhip().vkhip_kv_read(R(T.cache()), R(rows), T.A, T.A, T.A, T.A, None), "kv_read")


@pytest.mark.parametrize("change", [dict(o_row=0), dict(o_row=56), dict(o_head=0), dict(o_head=56), dict(o_row=256, o_head=256), dict(o_row=256, o_head=200)])
def test_kv_attention_refuses_output_rows_on_each_other(change):
    lib = V.vkhip()
    d = V.KvAttentionDesc(**{**dict(q_heads=4, q_tokens=1, dtype=0, scale=1.0, q_row=256, q_head=64, o_row=256, o_head=64), **change})
    T.refused(lib.vkhip_kv_attention(R(d), R(T.cache()), T.A, T.A, T.A, T.A, None), "kv_attention")
    assert lib.vkhip_kv_attention_workspace_bytes(R(d), R(T.cache())) == 0


def test_one_row_or_head_needs_no_stride():
    """Strides that are never taken may be 0: one row, one head."""
    lib = V.vkhip()
    many = dict(batch=1, q_heads=8, kv_heads=1, head_dim=64, dtype=0, causal=0, scale=0.1, q_head=64, k_row=64, v_row=64, total_k=100000)
    assert lib.vkhip_attention_workspace_bytes(R(V.AttentionDesc(**many, total_q=1, o_row=0, o_head=64))) > 0
    assert lib.vkhip_attention_workspace_bytes(R(V.AttentionDesc(**{**many, "q_heads": 1}, total_q=9, o_row=64, o_head=0))) > 0
    assert lib.vkhip_attention_workspace_bytes(R(V.AttentionDesc(**many, total_q=9, o_row=64, o_head=9 * 64))) > 0  # heads outside rows
