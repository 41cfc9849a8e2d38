"""Group norm, packed attention, the 8-bit cache's rows and the attention over it, against their
definitions in float64.

Tolerances follow from the roundings of each operator: u is half a step of the output type (2^-11 for
fp16, 2^-8 for bf16, whose next number after 1 is 1 + 2^-7, 2^-24 for fp32).
 * group norm: one rounding of y, and fp32 arithmetic on (x - mean) * rstd * gamma + beta, a few units of
   2^-24 of each term's size (16 of them allowed), the activation's hardware exp and reciprocal included.
   No activation has a slope above 1.2.
 * attention: weights p in [0, 1] are rounded once to the 16-bit type (their fp32 sum is not), which moves
   o by at most u_p * sum p|v|; scores are sums of D fp32 products, whose error e moves every weight by a
   factor of at most 1 + 2e; one rounding of o. fp16 weights below 2^-14 are off by up to 2^-25 each.
 * cache rows: s and x / s are fp32, so a stored byte may differ from the float64 one only where the
   quotient is within 127 * 2^-22 of a tie; values read back are one rounding of byte * scale.
"""
import ctypes
import math

import numpy as np
import pytest

import vknn_amd as V
from vknn_amd import DeviceBuffer, check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

DT = {"f16": (torch.float16, V.DT_F16, 2.0 ** -11), "bf16": (torch.bfloat16, V.DT_BF16, 2.0 ** -8), "f32": (torch.float32, V.DT_F32, 2.0 ** -24)}
TINY = {"f16": 2.0 ** -25, "bf16": 1e-38, "f32": 1e-38}


def rand(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


class Dev:
    """A CPU tensor's copy in device memory (torch computes on the CPU here: its own GPU runtime is not needed)."""

    def __init__(self, t):
        self.shape, self.dtype = t.shape, t.dtype
        self.nbytes = t.numel() * t.element_size()
        self.buf = DeviceBuffer(max(self.nbytes, 16))
        self.put(t)

    @classmethod
    def zeros(cls, shape, dtype):
        self = cls.__new__(cls)
        self.shape, self.dtype, self.nbytes = torch.Size(shape), dtype, math.prod(shape) * torch.empty(0, dtype=dtype).element_size()
        self.buf = DeviceBuffer(self.nbytes)
        self.buf.zero()
        return self

    def data_ptr(self):
        return self.buf.ptr

    def put(self, t):
        assert t.shape == self.shape and t.dtype == self.dtype
        if self.nbytes:
            self.buf.upload(t.contiguous().flatten().view(torch.uint8).numpy())

    def get(self):
        return torch.from_numpy(self.buf.download(np.uint8, self.nbytes)).view(self.dtype).view(self.shape)

    def rows(self, ids):
        """Some entries of the first axis, without the others."""
        each = self.nbytes // self.shape[0]
        out = np.empty((len(ids), each), np.uint8)
        for i, k in enumerate(ids):
            check(V.vkhip().vkhip_memcpy_d2h(out[i].ctypes.data, self.buf.ptr + int(k) * each, each, None), "d2h")
        return torch.from_numpy(out.reshape(-1)).view(self.dtype).view(len(ids), *self.shape[1:])


def full(shape, value, dtype):
    return Dev(torch.full(shape, value, dtype=dtype))


def ints(a):
    return Dev(torch.tensor(a, dtype=torch.int32))


def workspace(n):
    """Scratch with NaN bit patterns: what is read without being written shows."""
    return full((max(n, 16),), 255, torch.uint8)


def sync():
    check(V.vkhip().vkhip_device_sync(), "sync")


# ------------------------------------------------------------------------------------ group norm
def act64(z, act, lo, hi):
    return {0: lambda: z, 1: lambda: z.clamp(min=0), 2: lambda: z.clamp(0, 6), 3: lambda: z.clamp(lo, hi), 4: lambda: z * (z + 3).clamp(0, 6) / 6,
            5: lambda: z * torch.sigmoid(z), 6: lambda: (lo * z + hi).clamp(0, 1)}[act]()


def to_nc4(x):
    """[n, p, c] -> NC4HW4 [n, ceil(c/4), p, 4], missing channels zero."""
    n, p, c = x.shape
    y = torch.zeros((n, p, (c + 3) // 4 * 4), dtype=x.dtype)
    y[:, :, :c] = x
    return y.view(n, p, -1, 4).permute(0, 2, 1, 3).contiguous()


def from_nc4(y, c):
    return y.permute(0, 2, 1, 3).reshape(y.shape[0], y.shape[2], -1)[:, :, :c]


def group_norm(lib, x, groups, gamma, beta, dtype="f16", xf=1, yf=1, act=0, lo=0.0, hi=0.0, eps=1e-5, h=None, x_pad=0, y_pad=0, stream=None, inplace=False):
    """x: [n, p, c] CPU values of the type; the output [n, p, c], and what lay beside its rows."""
    n, p, c = x.shape
    dt, code, _ = DT[dtype]
    h = h or p
    if xf == 2:
        dx = Dev(to_nc4(x).to(dt))
    else:
        rows = torch.full((n, p, c + x_pad), float("nan"), dtype=dt)
        rows[:, :, :c] = x.to(dt)
        dx = Dev(rows)
    dy = dx if inplace else full((n, (c + 3) // 4, p, 4) if yf == 2 else (n, p, c + y_pad), 7.0, dt)
    d = V.GroupNormDesc(N=n, C=c, H=h, W=p // h, groups=groups, x_fmt=xf, y_fmt=yf, dtype=code, act=act, act_lo=lo, act_hi=hi, eps=eps,
                        x_row=c + x_pad if x_pad else 0, y_row=c + y_pad if y_pad else 0)
    ws = workspace(lib.vkhip_group_norm_workspace_bytes(ctypes.byref(d)))
    g, b = (None if t is None else Dev(t.float()) for t in (gamma, beta))
    sync()
    check(lib.vkhip_group_norm(ctypes.byref(d), dx.data_ptr(), None if g is None else g.data_ptr(), None if b is None else b.data_ptr(), dy.data_ptr(), ws.data_ptr(),
                               stream), "group_norm")
    sync()
    if yf == 2:
        y = dy.get().permute(0, 2, 1, 3).reshape(n, p, -1)
        assert (y[:, :, c:] == 0).all(), "channels past C are zero"
        return y[:, :, :c].double()
    y = dy.get()
    if not inplace:
        assert (y[:, :, c:] == 7.0).all(), "nothing beside the rows is written"
    return y[:, :, :c].double()


def check_gn(y, x, groups, gamma, beta, dtype, act, lo=0.0, hi=0.0, eps=1e-5):
    n, p, c = x.shape
    x = x.double().view(n, p, groups, c // groups)
    mean, var = x.mean((1, 3), keepdim=True), x.var((1, 3), keepdim=True, correction=0)
    rstd = 1 / (var + eps).sqrt()
    ga = torch.ones(c, dtype=torch.float64) if gamma is None else gamma.double()
    be = torch.zeros(c, dtype=torch.float64) if beta is None else beta.double()
    z = ((x - mean) * rstd).view(n, p, c) * ga + be
    want = act64(z, act, lo, hi)
    size = (((x - mean).abs() + mean.abs() + var.sqrt()) * rstd).view(n, p, c) * ga.abs() + be.abs()
    slope = max(1.2, abs(lo)) if act == 6 else 1.2
    bound = DT[dtype][2] * want.abs() * 1.01 + TINY[dtype] + 16 * 2.0 ** -24 * slope * (size + 1)
    worst = ((y - want).abs() / bound).max().item()
    assert worst <= 1, worst


GN_SIZES = [(1, 1, 4, 1), (1, 1, 6, 3), (2, 7, 20, 4), (1, 49, 32, 32), (3, 33, 36, 9), (1, 1600, 128, 32), (2, 35, 108, 27), (1, 300, 2056, 8), (65, 9, 16, 1), (1, 4099, 24, 2)]


@pytest.mark.parametrize("n,p,c,groups", GN_SIZES)
@pytest.mark.parametrize("dtype,xf,yf", [("f16", 1, 1), ("bf16", 1, 1), ("f32", 1, 1), ("f16", 2, 1), ("f16", 2, 2), ("f16", 1, 2)])
def test_group_norm(gpu, n, p, c, groups, dtype, xf, yf):
    act = (n + p + c) % 7
    lo, hi = (0.3, 0.4) if act == 6 else (-0.5, 0.8)
    x = (rand(p + c, n, p, c) * (1 + torch.arange(c) % 5) + torch.arange(c) % 3).to(DT[dtype][0]).float()
    gamma, beta = rand(1, c), rand(2, c)
    y = group_norm(V.vkhip(), x, groups, gamma, beta, dtype, xf, yf, act, lo, hi)
    check_gn(y, x, groups, gamma, beta, dtype, act, lo, hi)


@pytest.mark.parametrize("xf,yf,c,x_pad,y_pad", [(1, 1, 30, 0, 0), (1, 1, 13, 0, 0), (1, 1, 64, 8, 0), (1, 1, 64, 3, 5), (1, 1, 64, 0, 4), (1, 2, 13, 2, 0), (2, 1, 13, 0, 1),
                                                (2, 1, 16, 0, 3), (1, 2, 16, 4, 0), (2, 2, 5, 0, 0)])
def test_group_norm_rows_and_odd_channels(gpu, xf, yf, c, x_pad, y_pad):
    x = rand(c, 2, 77, c).half().float()
    beta = rand(3, c)
    groups = 1 if c in (13, 5) else 2
    y = group_norm(V.vkhip(), x, groups, None, beta, "f16", xf, yf, 5, x_pad=x_pad, y_pad=y_pad, h=7)
    check_gn(y, x, groups, None, beta, "f16", 5)


def test_group_norm_far_from_zero(gpu):
    """A mean of 2000 deviations: the difference of two sums would leave nothing of the variance."""
    x = (rand(5, 2, 900, 16) + 2000).float()
    check_gn(group_norm(V.vkhip(), x, 4, None, None, "f32"), x, 4, None, None, "f32", 0)
    x = torch.full((1, 500, 8), 3.0)  # no variance at all
    assert (group_norm(V.vkhip(), x, 2, None, rand(1, 8) * 0, "f32") == 0).all()


def test_group_norm_spoiled_image(gpu):
    """A NaN stays in its image and group; infinities past C in NC4HW4 are not part of it."""
    x = rand(6, 3, 50, 16).half().float()
    clean = group_norm(V.vkhip(), x, 4, None, None)
    bad = x.clone()
    bad[1, 7, 5] = float("nan")
    y = group_norm(V.vkhip(), bad, 4, None, None)
    assert torch.isnan(y[1, :, 4:8]).all()
    y[1, :, 4:8] = clean[1, :, 4:8]
    assert torch.equal(y, clean)


def test_group_norm_in_place_and_empty(gpu):
    lib, x = V.vkhip(), rand(7, 2, 130, 48).half().float()
    a = group_norm(lib, x, 6, None, None)
    assert torch.equal(a, group_norm(lib, x, 6, None, None, inplace=True))
    d = V.GroupNormDesc(N=0, C=8, H=4, W=4, groups=2, x_fmt=1, y_fmt=1, dtype=0)
    assert lib.vkhip_group_norm(ctypes.byref(d), None, None, None, None, None, None) == 0


# ------------------------------------------------------------------------------------ packed attention
def attention(lib, q, k, v, nq, nk, causal, dtype, scale, stream=None, joint=False, o_pad=0):
    """q [sum nq, hq, d], k, v [sum nk, hkv, d]; joint: the three are slices of one row matrix."""
    dt, code, _ = DT[dtype]
    hq, hkv, d = q.shape[1], k.shape[1], q.shape[2]
    if joint:
        rows = Dev(torch.cat([q.flatten(1), k.flatten(1), v.flatten(1)], 1).to(dt))
        width = (hq + 2 * hkv) * d
        ptr = [rows.data_ptr(), rows.data_ptr() + hq * d * 2, rows.data_ptr() + (hq + hkv) * d * 2]
        strides = [(width, d)] * 3
    else:  # heads outside rows
        held = [Dev(t.transpose(0, 1).contiguous().to(dt)) for t in (q, k, v)]
        ptr = [t.data_ptr() for t in held]
        strides = [(d, t.shape[0] * d) for t in (q, k, v)]
    out = full((q.shape[0], hq, d + o_pad), 7.0, dt)
    desc = V.AttentionDesc(batch=len(nq), q_heads=hq, kv_heads=hkv, head_dim=d, total_q=q.shape[0], total_k=k.shape[0], dtype=code, causal=int(causal), scale=scale,
                           q_row=strides[0][0], q_head=strides[0][1], k_row=strides[1][0], k_head=strides[1][1], v_row=strides[2][0], v_head=strides[2][1],
                           o_row=hq * (d + o_pad), o_head=d + o_pad)
    cq, ck = ints(np.cumsum([0] + list(nq)).tolist()), ints(np.cumsum([0] + list(nk)).tolist())
    ws = workspace(lib.vkhip_attention_workspace_bytes(ctypes.byref(desc)))
    sync()
    check(lib.vkhip_attention_packed(ctypes.byref(desc), *ptr, cq.data_ptr(), ck.data_ptr(), out.data_ptr(), ws.data_ptr(), stream),
          "attention_packed")
    sync()
    out = out.get()
    assert (out[:, :, d:] == 7.0).all()
    return out[:, :, :d].double()


def attention64(q, k, v, see, scale):
    """One head: o, the bound's terms sum p|v| and sum |q||k| scale; see: bool [nq, nk]. Unseen keys do not exist."""
    z = torch.where(see, q @ k.T * scale, -math.inf)
    p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
    return p @ v, p @ v.abs(), (q.abs() @ k.abs().T * scale).masked_fill(~see, 0).amax(1, keepdim=True)


def check_attention(out, q, k, v, nq, nk, causal, dtype, scale, weights_dtype=None, extra=0.0):
    hq, hkv = q.shape[1], k.shape[1]
    u, up = DT[dtype][2], DT[weights_dtype or dtype][2]
    a = b = 0
    for n, m in zip(nq, nk):
        see = torch.arange(m)[None] <= torch.arange(n)[:, None] + m - n if causal else torch.ones(n, m, dtype=torch.bool)
        for h in range(hq if n and m else 0):
            kk, vv = k[b:b + m, h * hkv // hq].double(), v[b:b + m, h * hkv // hq].double()
            want, pv, qk = attention64(q[a:a + n, h].double(), kk, vv, see, scale)
            e = (q.shape[2] + 16) * 2.0 ** -24 * qk + 2.0 ** -20 + extra * qk
            bound = u * want.abs() * 1.01 + TINY[dtype] + (up * 1.02 + 2 * e) * pv + m * 2.0 ** -25 * vv.abs().amax(0, keepdim=True)
            worst = ((out[a:a + n, h] - want).abs() / bound).max().item()
            assert worst <= 1, (worst, n, m, h)
        if n and not m:
            assert (out[a:a + n] == 0).all()
        a, b = a + n, b + m


def attention_inputs(seed, nq, nk, hq, hkv, d, dtype):
    dt = DT[dtype][0]
    return (rand(seed, sum(nq), hq, d).to(dt).float(), rand(seed + 1, sum(nk), hkv, d).to(dt).float(), rand(seed + 2, sum(nk), hkv, d).to(dt).float())


ATTN = [([1], [1]), ([1], [129]), ([3, 0, 1], [3, 5, 1]), ([128, 129], [128, 129]), ([63, 64, 65], [63, 64, 65]), ([200], [70]), ([5, 77], [600, 0]), ([300, 1, 31], [300, 400, 95]), ([257], [1024])]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("nq,nk", ATTN)
@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 64), (6, 2, 128), (3, 1, 40)])
def test_attention(gpu, dtype, causal, nq, nk, hq, hkv, d):
    q, k, v = attention_inputs(sum(nq) + d, nq, nk, hq, hkv, d, dtype)
    out = attention(V.vkhip(), q, k, v, nq, nk, causal, dtype, d ** -0.5, joint=sum(nq) == sum(nk))
    check_attention(out, q, k, v, nq, nk, causal, dtype, d ** -0.5)


@pytest.mark.parametrize("d", [8, 16, 24, 72, 80, 96, 104, 120])
def test_attention_head_dims(gpu, d):
    nq, nk = [70, 33], [70, 33]
    q, k, v = attention_inputs(d, nq, nk, 4, 2, d, "f16")
    check_attention(attention(V.vkhip(), q, k, v, nq, nk, True, "f16", d ** -0.5, joint=True, o_pad=8), q, k, v, nq, nk, True, "f16", d ** -0.5)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attention_large_scores(gpu, dtype):
    """Scores in the hundreds: a running maximum that grows late, rows that one key owns."""
    nq, nk = [150], [333]
    q, k, v = attention_inputs(3, nq, nk, 2, 1, 64, dtype)
    k = (k * torch.linspace(0.1, 8, 333)[:, None, None]).to(DT[dtype][0]).float()
    check_attention(attention(V.vkhip(), q, k, v, nq, nk, False, dtype, 1.0), q, k, v, nq, nk, False, dtype, 1.0)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attention_spoiled_rows_stay_unseen(gpu, dtype, bad):
    """Keys and values that are not finite reach the queries that see them and no other: neither earlier queries
    of the sequence nor the next one."""
    nq = [150, 40]
    q, k, v = attention_inputs(11, nq, nq, 2, 2, 128, dtype)
    clean = attention(V.vkhip(), q, k, v, nq, nq, True, dtype, 0.1)
    v2, k2 = v.clone(), k.clone()
    v2[100, :, 3] = bad
    k2[149, 0] = float("nan")
    v2[189] = bad  # the last row of all
    out = attention(V.vkhip(), q, k2, v2, nq, nq, True, dtype, 0.1)
    seen = torch.zeros(clean.shape, dtype=torch.bool)
    seen[100:150, :, 3] = True
    seen[149, 0] = True
    seen[189] = True
    assert torch.equal(out[~seen], clean[~seen])
    special = out[100:149, :, 3]
    assert torch.isnan(special).all() if math.isnan(bad) else (special == bad).all()
    assert torch.isnan(out[149, 0]).all()


def test_attention_both_infinities_make_nan(gpu):
    nq = [64]
    q, k, v = attention_inputs(12, nq, nq, 1, 1, 64, "f16")
    v[10, 0, 1], v[20, 0, 1], v[30, 0, 1] = float("inf"), float("-inf"), float("nan")
    out = attention(V.vkhip(), q, k, v, nq, nq, True, "f16", 0.1)[:, 0, 1]
    assert torch.isfinite(out[:10]).all() and (out[10:20] == float("inf")).all() and torch.isnan(out[20:]).all()


# ------------------------------------------------------------------------------------ the cache
class Cache:
    def __init__(self, batch, blocks, page, heads, d, seed=0, spare=3):
        self.page, self.heads, self.d, self.batch, self.blocks = page, heads, d, batch, blocks
        self.dp = V.vkhip().vkhip_kv_row(d)
        self.pages = batch * blocks + spare
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randperm(self.pages, generator=g)[:batch * blocks].view(batch, blocks).int()
        # what a recycled page holds: anything, scales not finite
        self.k = Dev(torch.randint(-128, 128, (self.pages, heads, page, self.dp), generator=g, dtype=torch.int8))
        self.v = Dev(torch.randint(-128, 128, (self.pages, heads, self.dp, page), generator=g, dtype=torch.int8))
        self.ks = full((self.pages, heads), float("nan"), torch.float32)
        self.vs = full((self.pages, heads), float("nan"), torch.float32)
        self.gpu_table = Dev(self.table)

    def desc(self):
        return V.KvCache(k=self.k.data_ptr(), v=self.v.data_ptr(), k_scale=self.ks.data_ptr(), v_scale=self.vs.data_ptr(), table=self.gpu_table.data_ptr(), pages=self.pages,
                         page_tokens=self.page, kv_heads=self.heads, head_dim=self.d, batch=self.batch, max_blocks=self.blocks)

    def rows(self, k, code):
        row, head = self.heads * k.shape[2], k.shape[2]
        return V.KvRows(dtype=code, total=k.shape[0], k_row=row, k_head=head, v_row=row, v_head=head)

    def append(self, k, v, new, lens, dtype, stream=None):
        dt, code, _ = DT[dtype]
        k, v = Dev(k.to(dt)), Dev(v.to(dt))
        cu, at = ints(np.cumsum([0] + list(new)).tolist()), ints(lens)
        sync()
        check(V.vkhip().vkhip_kv_append(ctypes.byref(self.desc()), ctypes.byref(self.rows(k, code)), k.data_ptr(), v.data_ptr(), cu.data_ptr(), at.data_ptr(), stream))
        sync()

    def read(self, start, count, dtype, pad=0):
        dt, code, _ = DT[dtype]
        k, v = (full((sum(count), self.heads, self.d + pad), 7.0, dt) for _ in range(2))
        cu, at = ints(np.cumsum([0] + list(count)).tolist()), ints(start)
        sync()
        check(V.vkhip().vkhip_kv_read(ctypes.byref(self.desc()), ctypes.byref(self.rows(k, code)), at.data_ptr(), cu.data_ptr(), k.data_ptr(), v.data_ptr(), None))
        sync()
        k, v = k.get(), v.get()
        assert (k[:, :, self.d:] == 7.0).all() and (v[:, :, self.d:] == 7.0).all()
        return k[:, :, :self.d], v[:, :, :self.d]

    def bytes_of(self, b, n):
        """The stored bytes [n, heads, d] of sequence b and each token's scale [n, heads], keys and values."""
        ids = self.table[b, :-(-n // self.page)].long()
        k = self.k.rows(ids).permute(0, 2, 1, 3).reshape(-1, self.heads, self.dp)[:n, :, :self.d]
        v = self.v.rows(ids).permute(0, 3, 1, 2).reshape(-1, self.heads, self.dp)[:n, :, :self.d]
        return [(x, s.rows(ids).repeat_interleave(self.page, 0)[:n]) for x, s in ((k, self.ks), (v, self.vs))]


def append64(q, s, x, n0, page):
    """The definition in float64 on one sequence: bytes q [n0, h, d], scales s [n0, h] (per token), rows x. Returns
    exact quotients (before rounding) and scales of all tokens."""
    n = n0 + x.shape[0]
    quot, scale = torch.zeros(n, *x.shape[1:], dtype=torch.float64), torch.zeros(n, x.shape[1], dtype=torch.float64)
    for lo in range(0, n, page):
        hi, mid = min(n, lo + page), min(max(n0, lo), min(n, lo + page))
        s0 = s[lo].double() if mid > lo else torch.zeros(x.shape[1], dtype=torch.float64)
        new = x[mid - n0:hi - n0].double()
        s1 = torch.maximum(s0, new.abs().amax((0, 2)) / 127) if hi > mid else s0
        scale[lo:hi] = s1
        div = torch.where(s1 > 0, s1, 1.0)[None, :, None]
        quot[lo:mid] = q[lo:mid].double() * (s0[None, :, None] / div)
        quot[mid:hi] = new / div
    return quot, scale


CACHE = [(32, 2, 64, "f16"), (64, 1, 128, "f16"), (64, 3, 40, "bf16"), (128, 2, 96, "f16"), (256, 1, 128, "bf16"), (32, 1, 8, "bf16")]


@pytest.mark.parametrize("page,heads,d,dtype", CACHE)
def test_append_and_read(gpu, page, heads, d, dtype):
    """Rows in several calls: an empty page, the middle of one, over its end, single rows, none; louder rows later,
    so that scales grow under tokens already there."""
    lens = [0, 0, 0, 0]
    c = Cache(4, 5, page, heads, d)
    seen = [[(torch.zeros(0, heads, d, dtype=torch.int8), torch.zeros(0, heads)) for _ in range(2)] for _ in range(4)]
    for step, new in enumerate([[1, page, 0, 3], [2, 1, 2 * page + 5, page - 3], [page, 0, 1, 1], [1, 1, 1, 2 * page + 1], [1, page // 2, 7, 0]]):
        k = (rand(step, sum(new), heads, d) * 2.0 ** step).to(DT[dtype][0]).float()
        v = (rand(step + 50, sum(new), heads, d) * 3.0 ** (step % 3)).to(DT[dtype][0]).float()
        if step == 1:
            k[:2], v[:2] = 0, 0  # rows of zeros
        c.append(k, v, new, lens, dtype)
        at = 0
        for b, n in enumerate(new):
            got = c.bytes_of(b, lens[b] + n)
            for which, x in enumerate((k, v)):
                quot, scale = append64(*seen[b][which], x[at:at + n], lens[b], page)
                q, s = got[which]
                assert torch.allclose(s.double(), scale, rtol=2.0 ** -23, atol=0)
                away = (q.double() - quot).abs()
                assert (away <= 0.5 + 127 * 2.0 ** -22).all()
                # nothing moves where the scale did not grow
                old, old_s = seen[b][which]
                same = (s[:lens[b]] == old_s)[:, :, None].expand_as(old)
                assert torch.equal(q[:lens[b]][same], old[same])
            seen[b] = got
            lens[b] += n
            at += n
    start, count = [0, 5, page - 1, 1], [lens[0], lens[1] - 5, 2, lens[3] - 1]
    k, v = c.read(start, count, dtype, pad=8)
    at = 0
    for b in range(4):
        for rows, (q, s) in zip((k, v), c.bytes_of(b, lens[b])):
            want = (q.float() * s[:, :, None]).to(DT[dtype][0])[start[b]:start[b] + count[b]]
            assert torch.equal(rows[at:at + count[b]], want)
        at += count[b]


def test_append_tiny_and_large_rows(gpu):
    """Scales near the ends of the number ranges."""
    for dtype, values in (("f16", [6e-8, 1e-6, 65504.0]), ("bf16", [1.2e-38, 1e-30, 3e38])):
        c = Cache(1, 1, 32, 1, 64)
        for i, x in enumerate(values):
            k = (rand(i, 2, 1, 64).clamp(-1, 1) * x).to(DT[dtype][0]).float()
            c.append(k, k, [2], [0], dtype)
            for q, s in c.bytes_of(0, 2):
                quot, scale = append64(q[:0], s[:0], k, 0, 32)
                assert torch.allclose(s.double(), scale, rtol=2.0 ** -20, atol=2e-45)
                assert ((q.double() - k.double() / s.double()[:, :, None]).abs() <= 0.5 + 127 * 2.0 ** -22).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_append_not_finite(gpu, bad):
    """Such a row makes its head's page NaN and nothing else, until the page begins anew."""
    c = Cache(1, 2, 32, 2, 64)
    k, v = rand(1, 40, 2, 64), rand(2, 40, 2, 64)
    k[5, 1, 3] = bad
    c.append(k, v, [40], [0], "f16")
    rk, rv = c.read([0], [40], "f16")
    assert torch.isnan(rk[:32, 1]).all() and torch.isfinite(rk[:32, 0]).all() and torch.isfinite(rk[32:]).all() and torch.isfinite(rv).all()
    c.append(k[:3], v[:3], [3], [0], "f16")
    assert torch.isfinite(c.read([0], [3], "f16")[0]).all()


def test_cache_blocks_without_memory(gpu):
    c = Cache(2, 3, 32, 1, 64)
    names = c.table.clone()
    names[0, 1], names[1, 0], names[1, 2] = -1, c.pages, 1 << 30
    c.gpu_table.put(names)
    before = [t.get() for t in (c.k, c.v, c.ks, c.vs)]
    k, v = rand(3, 160, 1, 64), rand(4, 160, 1, 64)
    c.append(k, v, [80, 80], [0, 0], "f16")
    used = {int(c.table[0, 0]), int(c.table[0, 2]), int(c.table[1, 1])}
    for was, now in zip(before, [t.get() for t in (c.k, c.v, c.ks, c.vs)]):
        for p in set(range(c.pages)) - used:
            assert torch.equal(was[p].nan_to_num(1.5), now[p].nan_to_num(1.5)) if was.is_floating_point() else torch.equal(was[p], now[p])
    rk, _ = c.read([0, 0], [80, 80], "f16")
    assert (rk[32:64] == 0).all() and (rk[80:112] == 0).all() and (rk[144:] == 0).all() and (rk[:32] != 0).any()
    # tokens past the table are dropped
    c.append(k[:40], v[:40], [20, 20], [90, 96], "f16")


# ------------------------------------------------------------------------------------ attention over the cache
def kv_attention(lib, c, q, lens, dtype, scale, max_len=0, stream=None, o_pad=0):
    """q [batch, t, heads, d]"""
    dt, code, _ = DT[dtype]
    dq = Dev(q.to(dt))
    b, t, hq, d = q.shape
    out = full((b, t, hq, d + o_pad), 7.0, dt)
    desc = V.KvAttentionDesc(q_heads=hq, q_tokens=t, dtype=code, max_len=max_len, scale=scale, q_row=hq * d, q_head=d, o_row=hq * (d + o_pad), o_head=d + o_pad)
    cd, n = c.desc(), ints(lens)
    ws = workspace(lib.vkhip_kv_attention_workspace_bytes(ctypes.byref(desc), ctypes.byref(cd)))
    sync()
    check(lib.vkhip_kv_attention(ctypes.byref(desc), ctypes.byref(cd), dq.data_ptr(), n.data_ptr(), out.data_ptr(), ws.data_ptr(), stream), "kv_attention")
    sync()
    out = out.get()
    assert (out[..., d:] == 7.0).all()
    return out[..., :d].double()


def filled(batch, lens, page, heads, d, seed=0, blocks=None):
    c = Cache(batch, blocks or max(1, -(-max(lens) // page)), page, heads, d, seed)
    k, v = rand(seed + 1, sum(lens), heads, d), rand(seed + 2, sum(lens), heads, d) * 2
    k *= 1 + torch.arange(sum(lens))[:, None, None] // 40 % 5  # pages of different scales
    if sum(lens):
        c.append(k, v, lens, [0] * batch, "f16")
    return c


def check_kv_attention(out, c, q, lens, dtype, scale):
    # bf16 queries are scaled by powers of two into fp16: elements under 2^-14 of a row's largest are off by up to
    # 2^-25 of it, which moves a score by that part of max|q| sum|k|, at most d times sum |q||k| / d
    t, d = q.shape[1], q.shape[3]
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        (kq, ks), (vq, vs) = c.bytes_of(b, n)
        k, v = kq.double() * ks.double()[:, :, None], vq.double() * vs.double()[:, :, None]
        check_attention(out[b], q[b].double(), k, v, [t], [n], True, dtype, scale, weights_dtype="f16", extra=0.0 if dtype == "f16" else d * 2.0 ** -25)


STEP = [([1], 1), ([65, 0, 3], 1), ([64, 63, 300], 1), ([2, 700], 5), ([1100], 3), ([31, 32, 33, 97], 2)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page", [32, 64, 128])
@pytest.mark.parametrize("lens,t", STEP)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (7, 1, 72)])
def test_kv_attention(gpu, dtype, page, lens, t, hq, hkv, d):
    c = filled(len(lens), lens, page, hkv, d, seed=d + t)
    q = rand(9, len(lens), t, hq, d).to(DT[dtype][0]).float()
    check_kv_attention(kv_attention(V.vkhip(), c, q, lens, dtype, d ** -0.5, o_pad=8), c, q, lens, dtype, d ** -0.5)


@pytest.mark.parametrize("t,hq,hkv", [(1, 16, 1), (1, 17, 1), (1, 48, 1), (16, 8, 1), (64, 2, 2), (33, 6, 2)])
@pytest.mark.parametrize("page", [32, 256])
def test_kv_attention_many_rows(gpu, t, hq, hkv, page):
    lens = [500, 40, 64]
    c = filled(3, lens, page, hkv, 128, seed=t)
    q = rand(10, 3, t, hq, 128).half().float()
    check_kv_attention(kv_attention(V.vkhip(), c, q, lens, "f16", 0.07), c, q, lens, "f16", 0.07)


def test_kv_attention_large_queries(gpu):
    """bf16 queries beyond fp16's range, and rows whose elements differ by many powers of two."""
    lens = [130, 90]
    c = filled(2, lens, 64, 2, 64, seed=4)
    q = (rand(11, 2, 1, 4, 64) * torch.tensor([1e-6, 1.0, 1e5, 1e9])[None, None, :, None]).bfloat16().float()
    q[0, 0, 0, :32] *= 1e6
    q = q.bfloat16().float()
    for scale in (1e-9, 1e-5, 1.0):
        check_kv_attention(kv_attention(V.vkhip(), c, q, lens, "bf16", scale), c, q, lens, "bf16", scale)


def test_kv_attention_spoiled_pages(gpu):
    """A page of NaN scale reaches only the queries that see it; blocks without memory are seen by none."""
    lens = [100, 100]
    c = filled(2, lens, 32, 1, 64, seed=5)
    q = rand(12, 2, 8, 2, 64)
    clean = kv_attention(V.vkhip(), c, q.half().float(), lens, "f16", 0.125)
    for scales in (c.ks, c.vs):
        spoiled = scales.get()
        spoiled[int(c.table[0, 3])] = float("nan")  # holds tokens 96 .. 99
        scales.put(spoiled)
    out = kv_attention(V.vkhip(), c, q.half().float(), lens, "f16", 0.125)
    assert torch.equal(out[0, :4], clean[0, :4]) and torch.isnan(out[0, 4:]).all() and torch.equal(out[1], clean[1])
    names = c.table.clone()
    names[0, 3], names[1, 1] = -1, c.pages + 5
    c.gpu_table.put(names)
    out = kv_attention(V.vkhip(), c, q.half().float(), lens, "f16", 0.125)
    assert torch.isfinite(out).all() and torch.equal(out[0, :4], clean[0, :4])
    (kq, ks), (vq, vs) = c.bytes_of(1, 100)
    keep = torch.ones(100, dtype=torch.bool)
    keep[32:64] = False
    k, v = (kq.double() * ks.double()[:, :, None])[keep], (vq.double() * vs.double()[:, :, None])[keep]
    check_attention(out[1], q[1].half().double(), k, v, [8], [68], True, "f16", 0.125)
    c.gpu_table.put(torch.full_like(c.table, -1))
    assert (kv_attention(V.vkhip(), c, q.half().float(), lens, "f16", 0.125) == 0).all()


def test_kv_attention_max_len_and_growth(gpu):
    """max_len sizes the launch and cuts longer sequences; a table wider than the sequences changes nothing."""
    lens = [333, 64]
    c = filled(2, lens, 64, 2, 128, seed=6, blocks=40)
    q = rand(13, 2, 1, 4, 128).half().float()
    for most in (0, 333, 500, 2560):
        check_kv_attention(kv_attention(V.vkhip(), c, q, lens, "f16", 0.09, max_len=most), c, q, lens, "f16", 0.09)
    out = kv_attention(V.vkhip(), c, q, [333, 64], "f16", 0.09, max_len=100)
    check_kv_attention(out, c, q, [100, 64], "f16", 0.09)


def test_kv_long_cache(gpu):
    """Pages past 2^31 bytes and a sequence of 70001 tokens."""
    page, heads, d = 64, 8, 128
    pages = (1 << 31) // (heads * page * d) + 1200
    lens, blocks = [70001], 1094
    c = Cache.__new__(Cache)
    c.page, c.heads, c.d, c.dp, c.batch, c.blocks, c.pages = page, heads, d, 128, 1, blocks, pages
    c.table = (pages - 1 - torch.arange(blocks)).view(1, blocks).int()
    c.gpu_table = Dev(c.table)
    c.k, c.v = Dev.zeros((pages, heads, page, d), torch.int8), Dev.zeros((pages, heads, d, page), torch.int8)
    c.ks, c.vs = Dev.zeros((pages, heads), torch.float32), Dev.zeros((pages, heads), torch.float32)
    k, v = rand(1, 70001, heads, d), rand(2, 70001, heads, d)
    c.append(k, v, lens, [0], "f16")
    rk, rv = c.read([69990], [11], "f16")
    ids, ks, vs = c.table[0].long(), c.ks.get(), c.vs.get()
    low = torch.ones(pages, dtype=torch.bool)
    low[ids] = False
    assert (ks[low] == 0).all() and (ks[ids] > 0).all()
    assert (rk.float() - k[69990:].half().float()).abs().max() <= 0.51 * ks[ids].max().item() + 1e-3
    assert (rv.float() - v[69990:].half().float()).abs().max() <= 0.51 * vs[ids].max().item() + 1e-3
    q = rand(3, 1, 1, 8, d).half().float()
    check_kv_attention(kv_attention(V.vkhip(), c, q, lens, "f16", 0.09), c, q, lens, "f16", 0.09)


# ------------------------------------------------------------------------------------ streams and graphs
def test_own_stream_and_graph_replay(gpu):
    """The whole chain on a stream of its own, eager and as a graph that is replayed with new contents."""
    lib = V.vkhip()
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    check(lib.vkhip_stream_create(ctypes.byref(s)))
    n, p, c, heads, d = 2, 96, 64, 2, 32
    x = full((n, c // 4, p, 4), 0.0, torch.float16)
    tok, att = (full((n * p, c), 0.0, torch.float16) for _ in range(2))
    step = full((n, 1, heads, d), 0.0, torch.float16)
    cache = Cache(n, 3, 32, heads, d)
    cu, zero, lens = ints([0, p, 2 * p]), ints([0, 0]), ints([p, p])
    gn = V.GroupNormDesc(N=n, C=c, H=8, W=12, groups=8, x_fmt=2, y_fmt=1, dtype=0, act=5, eps=1e-5)
    ad = V.AttentionDesc(batch=n, q_heads=heads, kv_heads=heads, head_dim=d, total_q=n * p, total_k=n * p, dtype=0, causal=1, scale=0.2, q_row=c, q_head=d, k_row=c, k_head=d,
                         v_row=c, v_head=d, o_row=c, o_head=d)
    rows = V.KvRows(dtype=0, total=n * p, k_row=c, k_head=d, v_row=c, v_head=d)
    kd = V.KvAttentionDesc(q_heads=heads, q_tokens=1, dtype=0, max_len=p, scale=0.2, q_row=c, q_head=d, o_row=c, o_head=d)
    cd, r = cache.desc(), ctypes.byref
    w1 = workspace(lib.vkhip_group_norm_workspace_bytes(r(gn)))
    w2 = workspace(lib.vkhip_attention_workspace_bytes(r(ad)))
    w3 = workspace(lib.vkhip_kv_attention_workspace_bytes(r(kd), r(cd)))

    def chain():
        check(lib.vkhip_group_norm(r(gn), x.data_ptr(), None, None, tok.data_ptr(), w1.data_ptr(), s))
        check(lib.vkhip_attention_packed(r(ad), tok.data_ptr(), tok.data_ptr(), tok.data_ptr(), cu.data_ptr(), cu.data_ptr(), att.data_ptr(), w2.data_ptr(), s))
        check(lib.vkhip_kv_append(r(cd), r(rows), tok.data_ptr(), tok.data_ptr(), cu.data_ptr(), zero.data_ptr(), s))
        check(lib.vkhip_kv_attention(r(kd), r(cd), att.data_ptr(), lens.data_ptr(), step.data_ptr(), w3.data_ptr(), s))

    sync()
    check(lib.vkhip_graph_begin(s))
    chain()
    check(lib.vkhip_graph_end(s, ctypes.byref(g)))
    for i in range(4):
        x.put(rand(i, *x.shape).half())
        got = []
        for how in ("eager", "graph"):
            for t in (tok, att, step):
                t.put(torch.full(t.shape, 9.0, dtype=t.dtype))
            sync()
            if how == "eager":
                chain()
            else:
                check(lib.vkhip_graph_launch(g, s))
            check(lib.vkhip_stream_sync(s))
            got.append([t.get() for t in (tok, att, step, cache.ks, cache.vs)])
        for a, b in zip(*got):
            assert torch.isfinite(a[:4]).all() and torch.equal(a.nan_to_num(5.5), b.nan_to_num(5.5))
    check(lib.vkhip_graph_destroy(g))
    check(lib.vkhip_stream_destroy(s))


@pytest.mark.parametrize("nq,nk,hq,hkv,d", [([200], [4200], 2, 1, 128), ([130, 3], [130, 5000], 2, 2, 64), ([1], [3001], 4, 4, 72), ([500], [3], 1, 1, 64), ([300, 0, 20], [2500, 7, 2048], 1, 1, 128)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_few_queries_many_keys(gpu, nq, nk, hq, hkv, d, causal):
    """Calls whose keys are split over workgroups (few queries and heads, 1024 keys or more each)."""
    d0 = V.AttentionDesc(batch=len(nq), q_heads=hq, kv_heads=hkv, head_dim=d, total_q=sum(nq), total_k=sum(nk), dtype=0, causal=int(causal), scale=0.1, q_row=hq * d, q_head=d,
                         k_row=hkv * d, k_head=d, v_row=hkv * d, v_head=d, o_row=hq * d, o_head=d)
    assert (V.vkhip().vkhip_attention_workspace_bytes(ctypes.byref(d0)) > 0) == (sum(nk) // len(nk) >= 2048)
    for dtype in ("f16", "bf16"):
        q, k, v = attention_inputs(sum(nq), nq, nk, hq, hkv, d, dtype)
        check_attention(attention(V.vkhip(), q, k, v, nq, nk, causal, dtype, d ** -0.5), q, k, v, nq, nk, causal, dtype, d ** -0.5)


def test_attention_many_sequences(gpu):
    """More sequences than a wave has lanes, lengths mixed with empty ones; and equal lengths."""
    r = np.random.default_rng(5)
    for lens in ([int(x) for x in r.integers(0, 300, 150)], [130] * 7, [1] * 200):
        q, k, v = attention_inputs(len(lens), lens, lens, 2, 1, 64, "f16")
        for causal in (True, False):
            check_attention(attention(V.vkhip(), q, k, v, lens, lens, causal, "f16", 0.125, joint=True), q, k, v, lens, lens, causal, "f16", 0.125)
