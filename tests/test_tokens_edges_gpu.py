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


# Weights far below a row's largest: fp16 holds them as multiples of 2^-24 (off by 2^-25 at most) of a reference. Where
# they are raised so that the largest is 2^up or more, that is 2^-(25 + up) of the largest.
def check_long_tail(out, q, k, v, scale, dtype, up):
    """All heads of one sequence on one key/value head, last query last; out, q [n, heads, d], k, v [m, d] float64."""
    n, m = q.shape[0], k.shape[0]
    see = torch.arange(m)[None] <= torch.arange(n)[:, None] + m - n
    u = T.DT[dtype][2]
    for h in range(q.shape[1]):
        want, pv, qk = T.attention64(q[:, h], k, v, see, scale)
        e = (q.shape[2] + 16) * 2.0 ** -24 * qk + 2.0 ** -20 + (0.0 if dtype == "f16" else q.shape[2] * 2.0 ** -25) * qk
        bound = u * want.abs() * 1.01 + T.TINY[dtype] + (2.0 ** -11 * 1.02 + 2 * e) * pv + m * 2.0 ** -(25 + up) * v.abs().amax(0, keepdim=True)
        worst = ((out[:, h] - want).abs() / bound).max().item()
        assert worst <= 1, (worst, h)


def long_tail_cache(n, page, d, at):
    """One sequence whose token `at` has a key that all the others are 2^25 or so below, and a value of zero."""
    c = T.Cache(1, -(-n // page), page, 1, d, seed=n)
    g = torch.Generator().manual_seed(n)
    k = torch.zeros(c.k.shape, dtype=torch.int8)
    v = torch.zeros(c.v.shape, dtype=torch.int8)
    ids = c.table[0].long()
    rows = torch.randint(-1, 2, (len(ids), page, d), generator=g, dtype=torch.int8)
    rows[at // page, at % page] = 127
    k[ids, 0, :, :d] = rows
    vals = torch.randint(60, 128, (len(ids), d, page), generator=g, dtype=torch.int8)
    vals[at // page, :, at % page] = 0
    v[ids, 0, :d] = vals
    c.k.put(k)
    c.v.put(v)
    c.ks.put(torch.full(c.ks.shape, 0.01))
    c.vs.put(torch.full(c.vs.shape, 0.02))
    return c


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,page,d,hq,t,at", [(150001, 64, 128, 4, 1, 0), (20000, 32, 64, 2, 1, 19000), (40000, 64, 64, 8, 3, 0), (70000, 128, 96, 20, 1, 69999), (500, 64, 128, 1, 1, 3)])
def test_kv_attention_long_tail(gpu, n, page, d, hq, t, at, dtype):
    """A key that owns a row, and a hundred thousand small weights that are the whole of the output."""
    c = long_tail_cache(n, page, d, at)
    q = (1 + 0.01 * T.rand(n, 1, t, hq, d)).to(T.DT[dtype][0]).float()
    scale = 25.2 / 1.44269504 / (127 * 0.01 * d)
    out = T.kv_attention(V.vkhip(), c, q, [n], dtype, scale)
    (kq, ks), (vq, vs) = c.bytes_of(0, n)
    check_long_tail(out[0], q[0].double(), (kq.double() * ks.double()[:, :, None])[:, 0], (vq.double() * vs.double()[:, :, None])[:, 0], scale, dtype, 14)


@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 23, 2.0 ** 25, 2.0 ** 26, 2.0 ** 27, 2.0 ** 28, 2.0 ** 40, 2.0 ** 60])
def test_kv_attention_huge_scores(gpu, size):
    """Scores whose last places are whole powers of two or more: the row is its largest key's, or two equal ones'."""
    d, n, page = 64, 200, 64
    for keys in ([57], [0], [199], [3, 150], [64, 65]):
        c = T.Cache(1, 4, page, 1, d, seed=1)
        k, v = torch.zeros(c.k.shape, dtype=torch.int8), torch.randint(-127, 128, c.v.shape, generator=torch.Generator().manual_seed(5), dtype=torch.int8)
        ids = c.table[0].long()
        k[ids, 0, :, 0] = 100
        for i in keys:
            k[ids[i // page], 0, i % page, 0] = 101
        c.k.put(k)
        c.v.put(v)
        c.ks.put(torch.full(c.ks.shape, size))
        c.vs.put(torch.ones(c.vs.shape))
        q = torch.zeros(1, 1, 2, d)
        q[..., 0] = 1
        out = T.kv_attention(V.vkhip(), c, q, [n], "f16", 1.0)
        rows = torch.stack([v[ids[i // page], 0, :, i % page].double() for i in keys])
        assert torch.equal(out[0, 0], rows.mean(0).expand(2, d)), (size, keys)


@pytest.mark.parametrize("nq,nk,hq,at,causal", [(1, 40000, 2, 0, 1), (130, 20000, 1, 0, 1), (3, 300, 300, 7, 0), (70, 9000, 520, 0, 0), (257, 3001, 1, 2990, 1)])
def test_attention_long_tail(gpu, nq, nk, hq, at, causal):
    """fp16 rows where one key of value zero owns each row and the small weights are the whole of the output; with the
    keys split and not."""
    d, heads = 64, min(hq, 3)
    q = (1 + 0.01 * T.rand(nk, nq, 1, d)).half().float().expand(nq, hq, d)
    k, v = (0.005 * T.rand(nk + 1, nk, d)).half().float(), (1 + 0.2 * T.rand(nk + 2, nk, d)).half().float()
    k[at], v[at] = 1, 0
    scale = 25.2 / 1.44269504 / d
    out = T.attention(V.vkhip(), q, k[:, None], v[:, None], [nq], [nk], causal, "f16", scale)
    assert torch.equal(out, out[:, :1].expand_as(out))
    if causal:
        check_long_tail(out[:, :heads], q[:, :heads].double(), k.double(), v.double(), scale, "f16", 7)
    else:  # every query sees every key, as if each were the last
        for i in range(0, nq, 23):
            check_long_tail(out[i:i + 1, :heads], q[i:i + 1, :heads].double(), k.double(), v.double(), scale, "f16", 7)


@pytest.mark.parametrize("dtype,size", [("f16", 2.0 ** 12), ("f16", 2.0 ** 13), ("f16", 2.0 ** 14), ("f16", 2.0 ** 15), ("bf16", 2.0 ** 14), ("bf16", 2.0 ** 20), ("bf16", 2.0 ** 40)])
@pytest.mark.parametrize("nk", [64, 150, 2304])
def test_attention_huge_scores(gpu, dtype, size, nk):
    """Scores of 2^30 to 2^86, whose neighbours in fp32 are whole numbers apart: a row is its largest key's value, or the
    mean of two equal ones' (exact but for the output's rounding and the weights': equal weights, rounded alike, over
    their unrounded sum)."""
    d, nq = 64, 130
    u = T.DT[dtype][2]
    for keys in ([nk // 2], [0], [nk - 1], [1, nk - 2]):
        q = torch.full((nq, 1, d), size)
        k = torch.full((nk, 1, d), size * 0.75)
        k -= size * 2.0 ** -6 * (torch.arange(nk) % 5)[:, None, None]
        k[keys] = size
        v = T.rand(nk, nk, 1, d).to(T.DT[dtype][0]).float()
        for causal in (False, True):
            out = T.attention(V.vkhip(), q, k, v, [nq], [nk], causal, dtype, 1.0)
            # queries that see all of `keys`
            seen = out[max(0, nq - nk + max(keys)):] if causal else out
            want = v[keys].double().mean(0)
            assert ((seen - want).abs() <= 1.01 * u * want.abs() + 1.02 * u * v[keys].double().abs().mean(0) + T.TINY[dtype]).all(), (keys, causal)


@pytest.mark.parametrize("c,groups,p", [(20, 4, 301), (64, 2, 6400), (7, 1, 900), (24, 1, 40000)])
def test_group_norm_far_out(gpu, c, groups, p):
    """Means whose square leaves fp32: the variance is about the mean, so the norm of such rows is in range."""
    x = T.rand(p, 2, p, c) * 1e16 + 3e19
    T.check_gn(T.group_norm(V.vkhip(), x, groups, None, None, "f32"), x, groups, None, None, "f32", 0)
    x = torch.full((1, p, c), -1.0 * 2 ** 66)
    x[:, :, : c // groups] = 2.0 ** 70
    y = T.group_norm(V.vkhip(), x, groups, None, None, "bf16")
    T.check_gn(y, x, groups, None, None, "bf16", 0)


def test_group_norm_many_workgroups(gpu):
    """More groups of images than a launch has work items in one dimension (65535 x 257 workgroups of 256 threads)."""
    n, c, groups = 65535, 1028, 257
    some = T.rand(1, 51, 1, c).half().float()
    x = some.repeat(1285, 1, 1)
    y = T.group_norm(V.vkhip(), x, groups, None, None, "f16", 2, 2)
    T.check_gn(y[:51], some, groups, None, None, "f16", 0)
    assert torch.equal(y, y[:51].repeat(1285, 1, 1))


@pytest.mark.parametrize("batch,heads", [(64, (1 << 18) + 64), (70001, 3)])
def test_attention_many_workgroups(gpu, batch, heads):
    """More tiles and heads than a launch has work items in one dimension, and more tiles than workgroups in the second:
    sequences of one token, each its own only key, so that every head gives that token's value."""
    lib, d = V.vkhip(), 8
    q, v = T.Dev(T.rand(1, batch, d).half()), T.rand(2, batch, d).half()
    dv, out = T.Dev(v), T.Dev.zeros((batch, heads, d), torch.float16)
    desc = V.AttentionDesc(batch=batch, q_heads=heads, kv_heads=1, head_dim=d, total_q=batch, total_k=batch, dtype=V.DT_F16, causal=1, scale=0.5, q_row=d, q_head=0,
                           k_row=d, k_head=d, v_row=d, v_head=d, o_row=heads * d, o_head=d)
    cu, ws = T.ints(list(range(batch + 1))), T.workspace(lib.vkhip_attention_workspace_bytes(R(desc)))
    T.sync()
    check(lib.vkhip_attention_packed(R(desc), q.data_ptr(), q.data_ptr(), dv.data_ptr(), cu.data_ptr(), cu.data_ptr(), out.data_ptr(), ws.data_ptr(), None))
    T.sync()
    assert torch.equal(out.get(), v[:, None].expand(batch, heads, d))


@pytest.mark.parametrize("page", [32, 256])
def test_append_many_blocks(gpu, page):
    """More blocks of rows than a launch has workgroups in one dimension: 2^30 rows (one, read again and again), of which
    only the last block's have a page."""
    total, d = 1 << 30, 8
    c = T.Cache(1, 1, page, 1, d)
    c.blocks = total // page
    names = torch.full((1, c.blocks), -1, dtype=torch.int32)
    names[0, -1] = c.pages - 1
    c.gpu_table = T.Dev(names)
    k, v = T.rand(1, 1, d).half(), T.rand(2, 1, d).half()
    dk, dv, cu, at = T.Dev(k), T.Dev(v), T.ints([0, total]), T.ints([0])
    rows = V.KvRows(dtype=V.DT_F16, total=total, k_row=0, k_head=d, v_row=0, v_head=d)
    T.sync()
    check(V.vkhip().vkhip_kv_append(R(c.desc()), R(rows), dk.data_ptr(), dv.data_ptr(), cu.data_ptr(), at.data_ptr(), None))
    T.sync()
    for x, cells, scales in ((k, c.k.get()[-1, 0, :, :d], c.ks.get()), (v, c.v.get()[-1, 0, :d].T, c.vs.get())):
        assert torch.isnan(scales[:-1]).all()
        quot, scale = T.append64(torch.zeros(0, 1, d), torch.zeros(0, 1), x[None], 0, page)
        assert torch.allclose(scales[-1].double(), scale[0], rtol=2.0 ** -23, atol=0)
        assert ((cells.double() - quot[0]).abs() <= 0.5 + 127 * 2.0 ** -22).all()


@pytest.mark.parametrize("page,heads,d,dtype", [(32, 3, 64, "f16"), (64, 2, 128, "bf16"), (128, 1, 72, "f16"), (256, 2, 40, "bf16"), (64, 5, 8, "f16")])
def test_append_few_rows_to_filled_pages(gpu, page, heads, d, dtype):
    """Four rows a sequence or fewer, onto pages that hold tokens: the middle of a word, the last place of a page, a new
    page, several rows of one sequence over a page's end; scales that grow under the old tokens and that do not."""
    lens = [3, 1, 13, page - 1, page, page + 5, 2 * page - 3, 0]
    c = T.Cache(8, 4, page, heads, d)
    seen = [[(torch.zeros(0, heads, d, dtype=torch.int8), torch.zeros(0, heads)) for _ in range(2)] for _ in range(8)]
    fill, held = list(lens), [0] * 8
    steps = [fill, [1] * 8, [1] * 8, [0, 9, 0, 1, 0, 0, 13, 4], [1, 1, 1, 1, 1, 1, 1, 0], [0, 0, 31, 0, 0, 0, 0, 1], [4] * 8]
    for step, new in enumerate(steps):
        assert step == 0 or sum(new) <= 4 * len(new)
        # louder at every other step, quieter between; one head much louder, so that only its scale grows
        size = torch.ones(heads, 1) * (1.0 if step % 2 else 0.25)
        size[step % heads] = 2.0 ** step
        k = (T.rand(step, sum(new), heads, d) * size).to(T.DT[dtype][0]).float()
        v = (T.rand(step + 50, sum(new), heads, d) * size.flip(0)).to(T.DT[dtype][0]).float()
        c.append(k, v, new, held, dtype)
        at = 0
        for b, n in enumerate(new):
            got = c.bytes_of(b, held[b] + n)
            for which, x in enumerate((k, v)):
                quot, scale = T.append64(*seen[b][which], x[at:at + n], held[b], page)
                q, s = got[which]
                assert torch.allclose(s.double(), scale, rtol=2.0 ** -23, atol=0)
                assert ((q.double() - quot).abs() <= 0.5 + 127 * 2.0 ** -22).all()
                old, old_s = seen[b][which]
                same = (s[:held[b]] == old_s)[:, :, None].expand_as(old)
                assert torch.equal(q[:held[b]][same], old[same])
            seen[b] = got
            held[b] += n
            at += n


@pytest.mark.parametrize("n,p,c,groups", [(1, 1301, 20, 4), (2, 7001, 12, 1), (3, 1301, 21, 7), (1, 2049, 10, 1), (2, 512, 44, 4), (1, 30000, 24, 2), (1, 48000, 8, 2)])
@pytest.mark.parametrize("xf,yf", [(2, 1), (2, 2), (1, 2)])
def test_group_norm_planes_of_several_chunks(gpu, monkeypatch, n, p, c, groups, xf, yf):
    """NC4HW4 norms that no workgroup holds: several chunks of pixels, whole batches and a remainder; what lies past the
    channels is NaN."""
    def planes(x):
        y = torch.full((x.shape[0], x.shape[1], (c + 3) // 4 * 4), float("nan"), dtype=x.dtype)
        y[:, :, :c] = x
        return y.view(*x.shape[:2], -1, 4).permute(0, 2, 1, 3).contiguous()

    monkeypatch.setattr(T, "to_nc4", planes)
    x = (T.rand(p + c, n, p, c) * (1 + torch.arange(c) % 5) + torch.arange(c) % 3).half().float()
    gamma, beta = T.rand(1, c), T.rand(2, c)
    y = T.group_norm(V.vkhip(), x, groups, gamma, beta, "f16", xf, yf, 5)
    T.check_gn(y, x, groups, gamma, beta, "f16", 5)
