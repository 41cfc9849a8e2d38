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


# n pairs (the most of an axis with spectra): the last one's frequency is theta^(-(n - 1) / n), here on both sides of 10^6
@pytest.mark.parametrize("sections,spectra,n", [((32, 0, 0, 0), 0, 32), ((8, 24, 0, 0), 0, 32), ((8, 24, 0, 0), 1, 24), ((2, 30, 0, 0), 1, 30), ((16, 16, 0, 0), 1, 16)])
def test_rotary_refuses_theta_of_large_frequencies(sections, spectra, n):
    change = dict(rows=0, sections=sections, spectra=spectra, axes=2)
    edge = 1e6 ** (-n / (n - 1))
    T.refused(S.rotary({**change, "theta": edge * (1 - 1e-9)}), "rotary")
    assert S.rotary({**change, "theta": edge * (1 + 1e-9)}) == 0
    for theta in (1e-20, 1e-300, 5e-324):
        T.refused(S.rotary({**change, "theta": theta}), "rotary")
        T.refused(S.rotary({**change, "theta": theta, "rows": 4}), "rotary")
    for theta in (1e-3, 0.5, 1.0, 1e29):
        assert S.rotary({**change, "theta": theta}) == 0


def test_rotary_takes_any_theta_beside_one_pair_an_axis_or_given_frequencies():
    assert S.rotary(dict(rows=0, rotary_dim=2, sections=(1, 0, 0, 0), theta=1e-20)) == 0
    assert S.rotary(dict(rows=0, rotary_dim=4, sections=(1, 1, 0, 0), spectra=1, theta=1e-20)) == 0
    freq = (S.D * 32)(*[0.5] * 32)
    assert S.rotary(dict(rows=0, theta=1e-20), freq=ctypes.addressof(freq)) == 0
