"""What the operators of a token step refuse (rotary positions, pages, shared prefixes, norms around a block), before any
device work: every call here returns VKHIP_ERR_INVALID with a message that names the operator."""
import ctypes
import math

import pytest

import test_tokens as T
import vknn_amd as V

R, A = ctypes.byref, T.A
D = ctypes.c_double


def refused(rc, name):
    T.refused(rc, name)


RO = dict(rows=4, q_heads=4, k_heads=2, head_dim=64, rotary_dim=64, dtype=0, neighbours=0, axes=2, sections=(16, 16, 0, 0), interleaved=0, spectra=0, theta=1e4, pos_axis=4,
          q_row=512, q_head=64, k_row=512, k_head=64, qo_row=256, qo_head=64, ko_row=128, ko_head=64)


def rotary(change, pos=A, freq=None, q=A, k=A, qo=A + 4096, ko=A + 8192):
    return V.vkhip().vkhip_rotary(R(V.RotaryDesc(**{**RO, **change})), pos, freq, q, k, qo, ko, None)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(q_heads=0), dict(k_heads=-1), dict(q_heads=70000), dict(head_dim=1), dict(head_dim=264, qo_head=264), dict(rotary_dim=0),
                                    dict(rotary_dim=63), dict(rotary_dim=66), dict(dtype=3), dict(dtype=-1), dict(axes=0), dict(axes=5), dict(sections=(16, 15, 0, 0)),
                                    dict(sections=(48, -16, 0, 0)), dict(axes=1), dict(theta=0.0), dict(theta=float("nan")), dict(theta=-1.0), dict(theta=float("inf")), dict(pos_axis=-1),
                                    dict(q_row=-8), dict(k_head=-64), dict(qo_row=0), dict(qo_row=192), dict(qo_head=56), dict(ko_row=64), dict(ko_head=0),
                                    dict(sections=(1 << 30, 1 << 30, 1 << 30, (1 << 30) + 32), axes=4)])
def test_rotary_refuses(change):
    refused(rotary(change), "rotary")


@pytest.mark.parametrize("change", [dict(pos=None), dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(pos=A + 2), dict(q=A + 1), dict(ko=A + 8193), dict(qo=A), dict(ko=A)])
def test_rotary_refuses_pointers(change):
    refused(rotary({}, **change), "rotary")


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 1e6])
def test_rotary_refuses_frequencies(bad):
    freq = (D * 32)(*([0.5] * 31 + [bad]))
    refused(rotary({}, freq=ctypes.addressof(freq)), "rotary")


PAGES = dict(pages=8, page_tokens=64, kv_heads=1, head_dim=64, batch=2, max_blocks=4, table=A)


def reserve(cache={}, pool={}, total=4, lens=A, add=A + 16, cu=A + 32, now=A + 48, pos=A, slot=A):
    return V.vkhip().vkhip_kv_reserve(R(V.KvCache(**{**PAGES, **cache})), R(V.KvPool(**{**dict(free=A, state=A, capacity=8), **pool})), lens, add, total, cu, now, pos, slot, None)


def release(cache={}, pool={}, lens=A, keep=A + 16):
    return V.vkhip().vkhip_kv_release(R(V.KvCache(**{**PAGES, **cache})), R(V.KvPool(**{**dict(free=A, state=A, capacity=8), **pool})), lens, keep, None)


BAD_PAGES = [dict(cache=dict(pages=-1)), dict(cache=dict(page_tokens=48)), dict(cache=dict(batch=-1)), dict(cache=dict(batch=70000)), dict(cache=dict(max_blocks=-1)), dict(cache=dict(max_blocks=1 << 26)),
             dict(cache=dict(batch=65535, max_blocks=1 << 16)), dict(cache=dict(table=None)), dict(cache=dict(table=A + 2)), dict(pool=dict(capacity=-1)), dict(pool=dict(free=None)), dict(pool=dict(state=None)),
             dict(pool=dict(state=A + 1)), dict(pool=dict(free=A + 2)), dict(lens=None), dict(lens=A + 3)]


@pytest.mark.parametrize("change", BAD_PAGES)
def test_pages_refuse(change):
    refused(reserve(**change), "kv_reserve")
    refused(release(**change), "kv_release")


@pytest.mark.parametrize("change", [dict(total=-1), dict(total=1 << 30), dict(add=None), dict(cu=None), dict(cu=A + 2), dict(now=A + 1), dict(pos=A + 2), dict(slot=A + 4), dict(now=A), dict(cu=A),
                                    dict(cu=A + 16), dict(now=A + 16)])
def test_reserve_refuses(change):
    refused(reserve(**change), "kv_reserve")


def test_release_refuses():
    refused(release(keep=None), "kv_release")
    refused(release(keep=A + 1), "kv_release")


SH = dict(q_heads=4, q_tokens=1, dtype=0, scale=1.0, q_row=256, q_head=64, o_row=256, o_head=64)


def shared(desc={}, cache={}, prefix={}, q=A, lens=A, o=A, ws=A):
    p = V.KvPrefix(**{**dict(cu=A, tokens=A, groups=1, max_tokens=0, max_tail=0), **prefix})
    d, c, lib = V.KvAttentionDesc(**{**SH, **desc}), T.cache(**cache), V.vkhip()
    return lib.vkhip_kv_attention_shared(R(d), R(c), R(p), q, lens, o, ws, None), lib.vkhip_kv_attention_shared_workspace_bytes(R(d), R(c), R(p))


@pytest.mark.parametrize("change", [dict(q_heads=0), dict(q_heads=3), dict(q_tokens=0), dict(q_tokens=65), dict(dtype=2), dict(scale=0.0), dict(scale=float("nan")), dict(max_len=-1), dict(q_row=4),
                                    dict(o_head=-8), dict(o_row=0), dict(o_head=56)])
def test_shared_refuses(change):
    rc, size = shared(desc=change)
    refused(rc, "kv_attention_shared")
    assert size == 0


@pytest.mark.parametrize("change", T.CACHES)
def test_shared_refuses_caches(change):
    refused(shared(cache=change)[0], "kv_attention_shared")


@pytest.mark.parametrize("change", [dict(groups=-1), dict(groups=70000), dict(max_tokens=-1), dict(max_tail=-1)])
def test_shared_refuses_groups(change):
    rc, size = shared(prefix=change)
    refused(rc, "kv_attention_shared")
    assert size == 0


@pytest.mark.parametrize("change", [dict(prefix=dict(cu=None)), dict(prefix=dict(tokens=None)), dict(prefix=dict(cu=A + 2)), dict(prefix=dict(tokens=A + 1)), dict(q=None), dict(lens=None), dict(o=None),
                                    dict(q=A + 8), dict(o=A + 2), dict(lens=A + 2), dict(ws=None), dict(ws=A + 8)])
def test_shared_refuses_pointers(change):
    refused(shared(**change)[0], "kv_attention_shared")


def test_shared_workspace_holds_what_a_call_without_groups_takes():
    """Nothing to share: the call is kv_attention's, and so is the workspace."""
    lib, d, c = V.vkhip(), V.KvAttentionDesc(**SH), T.cache(max_blocks=4000)
    alone = lib.vkhip_kv_attention_workspace_bytes(R(d), R(c))
    assert alone > 0
    for p in (V.KvPrefix(groups=0), V.KvPrefix(cu=A, tokens=A, groups=1, max_tokens=63)):
        assert lib.vkhip_kv_attention_shared_workspace_bytes(R(d), R(c), R(p)) == alone


RN = dict(rows=4, dim=64, dtype=0, post=1, pre=2, mods=2, mod_rows=2, alpha=1.0, post_eps=1e-5, pre_eps=1e-5, x_row=64, r_row=64, h_row=64, y_row=64, mod_row=64)


def norm(change={}, x=A, r=A + 4096, post_w=None, post_b=None, gate=None, pre_w=None, pre_b=None, scale=None, shift=None, mod=None, h=A + 8192, y=A + 16384):
    return V.vkhip().vkhip_residual_norm(R(V.ResidualNormDesc(**{**RN, **change})), x, r, post_w, post_b, gate, pre_w, pre_b, scale, shift, mod, h, y, None)


@pytest.mark.parametrize("change", [dict(rows=-1), dict(dim=0), dict(dim=32769), dict(dtype=3), dict(dtype=-1), dict(post=3), dict(pre=-1), dict(post_eps=-1.0), dict(pre_eps=float("nan")),
                                    dict(pre_eps=float("inf")), dict(alpha=float("nan")), dict(alpha=float("inf")), dict(x_row=-64), dict(r_row=-1), dict(mod_row=-1), dict(mods=-1), dict(mod_rows=-1),
                                    dict(h_row=63), dict(y_row=0)])
def test_residual_norm_refuses(change):
    refused(norm(change), "residual_norm")


@pytest.mark.parametrize("change", [dict(x=None, r=None), dict(h=None, y=None), dict(x=A + 1), dict(r=A + 3), dict(h=A + 1), dict(y=A + 1), dict(post_w=A + 2), dict(pre_b=A + 1), dict(gate=A + 1),
                                    dict(gate=A, mod=A + 2), dict(h=A + 16384)])
def test_residual_norm_refuses_pointers(change):
    refused(norm(**change), "residual_norm")


@pytest.mark.parametrize("change", [dict(mods=0), dict(mods=1), dict(mod_rows=0), dict(mod_rows=1)])
def test_residual_norm_refuses_rows_without_a_vector(change):
    for vector in ("gate", "scale", "shift"):
        refused(norm(change, **{vector: A}), "residual_norm")


@pytest.mark.parametrize("change,where", [(dict(h_row=128), dict(h=A)), (dict(y_row=128), dict(y=A + 4096)), (dict(r_row=72), dict(h=A + 4096))])
def test_residual_norm_refuses_in_place_with_other_rows(change, where):
    refused(norm(change, **where), "residual_norm")


def test_nothing_to_do_is_fine():
    assert rotary(dict(rows=0), pos=None, q=None, k=None, qo=None, ko=None) == 0
    assert reserve(cache=dict(batch=0), lens=None, add=None, cu=None) == 0 and release(cache=dict(batch=0), lens=None, keep=None) == 0
    assert shared(cache=dict(batch=0))[0] == 0
    assert norm(dict(rows=0), x=None, r=None, h=None, y=None) == 0
    assert math.isfinite(V.RotaryDesc().theta)
