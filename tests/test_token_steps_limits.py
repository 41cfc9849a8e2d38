"""Sizes and arguments at the limits of the operators of a token step, without a device: what is refused and what is taken,
beside test_token_steps.py."""
import ctypes

import pytest

import test_token_steps as S
import test_tokens as T
import vknn_amd as V

R = ctypes.byref


def desc(q_heads, q_tokens, d):
    return dict(q_heads=q_heads, q_tokens=q_tokens, q_row=q_heads * d, q_head=d, o_row=q_heads * d, o_head=d)


@pytest.mark.parametrize("q_heads,q_tokens,batch", [(1024, 64, 65535), (2048, 64, 16384), (32768 + 1024, 64, 1)])
def test_shared_refuses_more_rows_than_a_launch(q_heads, q_tokens, batch):
    """Past 2^31 rows of a head, or 65535 blocks of heads and rows: refused, and no workspace is named."""
    rc, size = S.shared(desc=desc(q_heads, q_tokens, 8), cache=dict(kv_heads=1, head_dim=8, batch=batch, max_blocks=4))
    T.refused(rc, "kv_attention_shared")
    assert size == 0


@pytest.mark.parametrize("q_heads,q_tokens,batch,groups", [(1, 32, 32000, 34000), (8, 64, 16000, 2000), (1, 1, 65535, 65535), (1024, 64, 8, 8)])
def test_shared_takes_many_groups(q_heads, q_tokens, batch, groups):
    """More blocks of rows than a grid's third dimension holds."""
    lib, c = V.vkhip(), T.cache(kv_heads=1, head_dim=8, batch=batch, max_blocks=4)
    d = V.KvAttentionDesc(**{**S.SH, **desc(q_heads, q_tokens, 8)})
    assert lib.vkhip_kv_attention_shared_workspace_bytes(R(d), R(c), R(V.KvPrefix(cu=T.A, tokens=T.A, groups=groups))) > 0
