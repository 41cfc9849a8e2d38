"""The token operators at their edges: rows that belong to no sequence, scores and weights at the ends of the number
ranges, launches at the limits of a grid. Against float64, with the bounds of test_tokens_gpu.py."""
import ctypes

import pytest

import test_tokens_gpu as T
import vknn_amd as V
from vknn_amd import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
R = ctypes.byref


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk,split", [([20, 0, 9], [4100, 3, 2500], True), ([3], [2049], True), ([20, 0, 9], [40, 3, 25], False), ([140], [150], False)])
def test_attention_rows_outside_every_sequence(gpu, nq, nk, split, causal):
    """Query rows in front of the first sequence and behind the last stay as they are, bit for bit, whether or not the
    call splits its keys; the sequences' rows are what they are without the others."""
    lib, hq, hkv, d, front, behind = V.vkhip(), 2, 1, 64, 7, 130
    q, k, v = T.attention_inputs(sum(nk), nq, nk, hq, hkv, d, "f16")
    rows = front + sum(nq) + behind
    whole = torch.full((rows, hq, d), float("nan"))
    whole[front:front + sum(nq)] = q
    dq, dk, dv = (T.Dev(t.half()) for t in (whole, k, v))
    was = torch.arange(rows * hq * d).remainder(1999).half().view(rows, hq, d)
    out = T.Dev(was)
    desc = V.AttentionDesc(batch=len(nq), q_heads=hq, kv_heads=hkv, head_dim=d, total_q=rows, total_k=sum(nk), dtype=V.DT_F16, causal=int(causal), scale=d ** -0.5,
                           q_row=hq * d, q_head=d, k_row=hkv * d, k_head=d, v_row=hkv * d, v_head=d, o_row=hq * d, o_head=d)
    size = lib.vkhip_attention_workspace_bytes(R(desc))
    assert (size > 0) == split
    at = [front]
    for n in nq:
        at.append(at[-1] + n)
    cq, ck, ws = T.ints(at), T.ints([0] + torch.tensor(nk).cumsum(0).tolist()), T.workspace(size)
    T.sync()
    check(lib.vkhip_attention_packed(R(desc), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), cq.data_ptr(), ck.data_ptr(), out.data_ptr(), ws.data_ptr(), None))
    T.sync()
    got = out.get()
    outside = torch.ones(rows, dtype=torch.bool)
    outside[front:front + sum(nq)] = False
    assert torch.equal(got[outside], was[outside])
    T.check_attention(got[~outside].double(), q, k, v, nq, nk, causal, "f16", d ** -0.5)
