"""What the token operators refuse, before any device work: every call here returns VKHIP_ERR_INVALID with a
message that names the operator, and a refused descriptor has no workspace."""
import ctypes

import pytest

import vknn_amd as V

R = ctypes.byref
BUF = ctypes.create_string_buffer(256)
A = (ctypes.addressof(BUF) + 31) // 32 * 32  # an aligned host address: never dereferenced


def refused(rc, name):
    assert rc == 1
    assert V.vkhip().vkhip_last_error().decode().startswith(name + ":")


GN = dict(N=1, C=32, H=4, W=4, groups=8, x_fmt=1, y_fmt=1, dtype=0, act=0, eps=1e-5)


@pytest.mark.parametrize("change", [dict(C=0), dict(C=30), dict(groups=0), dict(N=-1), dict(H=-2), dict(N=70000), dict(C=8192), dict(H=1 << 16, W=1 << 16), dict(x_fmt=0), dict(y_fmt=3),
                                    dict(x_fmt=2, dtype=1), dict(y_fmt=2, dtype=2), dict(dtype=3), dict(dtype=-1), dict(act=7), dict(act=-1), dict(eps=-1.0),
                                    dict(eps=float("nan")), dict(x_row=31), dict(y_row=8)])
def test_group_norm_refuses(change):
    lib, d = V.vkhip(), V.GroupNormDesc(**{**GN, **change})
    refused(lib.vkhip_group_norm(R(d), A, None, None, A, A, None), "group_norm")
    assert lib.vkhip_group_norm_workspace_bytes(R(d)) == 0


@pytest.mark.parametrize("x,gamma,y,ws", [(None, None, A, A), (A, None, None, A), (A, None, A, None), (A + 1, None, A, A), (A, A + 2, A, A), (A, None, A + 1, A), (A, None, A, A + 8)])
def test_group_norm_refuses_pointers(x, gamma, y, ws):
    refused(V.vkhip().vkhip_group_norm(R(V.GroupNormDesc(**GN)), x, gamma, None, y, ws, None), "group_norm")


AT = dict(batch=1, q_heads=4, kv_heads=2, head_dim=64, total_q=8, total_k=8, dtype=0, causal=1, scale=0.125, q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64,
          o_row=256, o_head=64)


@pytest.mark.parametrize("change", [dict(batch=-1), dict(q_heads=0), dict(q_heads=3), dict(kv_heads=0), dict(head_dim=0), dict(head_dim=60), dict(head_dim=136), dict(total_q=-1),
                                    dict(total_k=-1), dict(dtype=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q_row=252),
                                    dict(k_head=4), dict(v_row=-128), dict(o_head=1), dict(k_row=1 << 24), dict(total_q=1 << 30, q_heads=1 << 10)])
def test_attention_refuses(change):
    d = V.AttentionDesc(**{**AT, **change})
    refused(V.vkhip().vkhip_attention_packed(R(d), A, A, A, A, A, A, A, None), "attention_packed")
    assert V.vkhip().vkhip_attention_workspace_bytes(R(d)) == 0


@pytest.mark.parametrize("at", range(6))
def test_attention_refuses_pointers(at):
    for bad in (None, A + 2):
        p = [A] * 6
        p[at] = bad
        refused(V.vkhip().vkhip_attention_packed(R(V.AttentionDesc(**AT)), *p, A, None), "attention_packed")


@pytest.mark.parametrize("change", [dict(k_row=56), dict(v_row=0)])
def test_attention_refuses_overlapping_rows(change):
    refused(V.vkhip().vkhip_attention_packed(R(V.AttentionDesc(**{**AT, **change})), A, A, A, A, A, A, A, None), "attention_packed")


def cache(**change):
    return V.KvCache(**{**dict(k=A, v=A, k_scale=A, v_scale=A, table=A, pages=8, page_tokens=64, kv_heads=2, head_dim=64, batch=2, max_blocks=4), **change})


CACHES = [dict(pages=-1), dict(page_tokens=16), dict(page_tokens=0), dict(page_tokens=96), dict(page_tokens=512), dict(kv_heads=0), dict(head_dim=4), dict(head_dim=65),
          dict(head_dim=256), dict(batch=-1), dict(batch=70000), dict(max_blocks=-1), dict(max_blocks=1 << 28), dict(k=None), dict(v=A + 8), dict(k_scale=None), dict(v_scale=A + 2),
          dict(table=None)]


@pytest.mark.parametrize("change", CACHES)
def test_cache_refused(change):
    lib, c = V.vkhip(), cache(**change)
    rows = V.KvRows(dtype=0, total=4, k_row=128, k_head=64, v_row=128, v_head=64)
    d = V.KvAttentionDesc(q_heads=2, q_tokens=1, dtype=0, scale=1.0, q_row=128, q_head=64, o_row=128, o_head=64)
    refused(lib.vkhip_kv_append(R(c), R(rows), A, A, A, A, None), "kv_append")
    refused(lib.vkhip_kv_read(R(c), R(rows), A, A, A, A, None), "kv_read")
    refused(lib.vkhip_kv_attention(R(d), R(c), A, A, A, A, None), "kv_attention")


@pytest.mark.parametrize("change", [dict(dtype=2), dict(total=-1), dict(k_row=4), dict(v_head=-8), dict(k_head=1)])
def test_rows_refused(change):
    lib = V.vkhip()
    rows = V.KvRows(**{**dict(dtype=0, total=4, k_row=128, k_head=64, v_row=128, v_head=64), **change})
    refused(lib.vkhip_kv_append(R(cache()), R(rows), A, A, A, A, None), "kv_append")
    refused(lib.vkhip_kv_read(R(cache()), R(rows), A, A, A, A, None), "kv_read")


@pytest.mark.parametrize("change", [dict(q_heads=0), dict(q_heads=3), dict(q_tokens=0), dict(q_tokens=65), dict(dtype=2), dict(scale=0.0), dict(scale=float("nan")), dict(max_len=-1),
                                    dict(q_row=4), dict(o_head=-8), dict(q_heads=1 << 17)])
def test_kv_attention_refuses(change):
    lib = V.vkhip()
    d = V.KvAttentionDesc(**{**dict(q_heads=4, q_tokens=1, dtype=0, scale=1.0, q_row=256, q_head=64, o_row=256, o_head=64), **change})
    refused(lib.vkhip_kv_attention(R(d), R(cache()), A, A, A, A, None), "kv_attention")
    assert lib.vkhip_kv_attention_workspace_bytes(R(d), R(cache())) == 0


def test_nothing_to_do_is_fine():
    lib = V.vkhip()
    d = V.AttentionDesc(**{**AT, "total_q": 0})
    assert lib.vkhip_attention_packed(R(d), None, None, None, None, None, None, None, None) == 0
    rows = V.KvRows(dtype=0, total=0, k_row=128, k_head=64, v_row=128, v_head=64)
    assert lib.vkhip_kv_append(R(cache()), R(rows), None, None, None, None, None) == 0
    assert [lib.vkhip_kv_row(d) for d in (8, 64, 72, 128, 0, 12, 136)] == [64, 64, 128, 128, 0, 0, 0]
