"""The operators of a token step against their definitions in float64 (positions' angles in 128 bits).

Tolerances, u half a step of the output type as in test_tokens_gpu.py:
 * rotary: the angle's fraction of a turn is off by 2^-33 and by what position * 2^-65 adds; its sine and cosine are a
   handful of fp32 operations, 4 * 2^-24 allowed, and each of the two products and their sum is rounded once: 8 * 2^-24 of
   |a cos| + |b sin| <= |a| + |b|, and one rounding of the output.
 * pages: whole numbers, equal.
 * shared prefixes: the bounds of test_tokens_gpu.py's attention over the cache; parts are joined in fp32.
 * norms: a sum of n terms of one sign, at most 32 in a thread and then by halves, is off by (32 + log2 n) 2^-24 of itself,
   fp32 arithmetic by a few units of 2^-24 of each term's size: 64 of them allowed for a norm. What N_pre's input is off by
   passes through it, multiplied by rstd w, itself and by way of mean and deviation.
"""
import ctypes
import math
from decimal import Decimal, localcontext

import numpy as np
import pytest

import test_tokens_gpu as T
import vknn_amd as V
from test_tokens_gpu import DT, TINY, Dev, full, ints, rand, sync, workspace
from vknn_amd import check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
R = ctypes.byref
F32 = 2.0 ** -24


# ------------------------------------------------------------------------------------ rotary positions
def pairs_of(sections, interleaved):
    """(axis, number within the axis) of each pair."""
    left, had, got = list(sections), [0] * len(sections), []
    while any(left):
        for a in range(len(left)):
            for _ in range(min(left[a], 1) if interleaved else left[a]):
                got.append((a, had[a]))
                left[a], had[a] = left[a] - 1, had[a] + 1
    return got


def rotary(q, k, pos, sections, rot=None, dtype="f16", near=False, interleaved=False, spectra=False, theta=1e4, freq=None, layout="slices", stream=None):
    """q [rows, hq, d], k [rows, hk, d] or None, pos [axes, rows] -> the turned ones. layout: slices of one row matrix into
    tensors of their own, heads outside rows, or in place; `pad` values beside the rows stay."""
    lib, (dt, code, _) = V.vkhip(), DT[dtype]
    rows, hq, d = q.shape
    hk = 0 if k is None else k.shape[1]
    rot = rot or d
    size = torch.empty(0, dtype=dt).element_size()
    if layout == "heads":
        dq, dk = Dev(q.transpose(0, 1).contiguous().to(dt)), Dev(k.transpose(0, 1).contiguous().to(dt)) if hk else None
        ptr, strides = (dq.data_ptr(), dk.data_ptr() if hk else None), [(d, rows * d)] * 2
    else:
        pad = 8 if layout != "odd" else 3
        joint = Dev(torch.cat([q.flatten(1)] + ([k.flatten(1)] if hk else []) + [torch.full((rows, pad), 5.0)], 1).to(dt))
        width = (hq + hk) * d + pad
        ptr, strides = (joint.data_ptr(), joint.data_ptr() + hq * d * size), [(width, d)] * 2
    if layout == "place":
        optr, ostr = ptr, strides
    else:
        oq, ok = full((rows, hq, d + 8), 7.0, dt), full((rows, max(hk, 1), d + 8), 7.0, dt)
        optr, ostr = (oq.data_ptr(), ok.data_ptr()), [(hq * (d + 8), d + 8), (hk * (d + 8), d + 8)]
    dp = Dev(torch.from_numpy(np.ascontiguousarray(pos, dtype=np.int32)))
    desc = V.RotaryDesc(rows=rows, q_heads=hq, k_heads=hk, head_dim=d, rotary_dim=rot, dtype=code, neighbours=int(near), axes=len(sections), sections=tuple(list(sections) + [0] * (4 - len(sections))),
                        interleaved=int(interleaved), spectra=int(spectra), theta=theta, pos_axis=rows, q_row=strides[0][0], q_head=strides[0][1], k_row=strides[1][0], k_head=strides[1][1],
                        qo_row=ostr[0][0], qo_head=ostr[0][1], ko_row=ostr[1][0], ko_head=ostr[1][1])
    host = None if freq is None else (ctypes.c_double * len(freq))(*freq)
    sync()
    check(lib.vkhip_rotary(R(desc), dp.data_ptr(), None if host is None else ctypes.addressof(host), ptr[0], ptr[1] if hk else None, optr[0], optr[1] if hk else None, stream), "rotary")
    sync()
    if layout == "place":
        out = joint.get()
        assert (out[:, (hq + hk) * d:] == 5.0).all()
        return out[:, :hq * d].view(rows, hq, d), out[:, hq * d:(hq + hk) * d].view(rows, hk, d) if hk else None
    for o, n in ((oq, hq), (ok, hk)):
        assert (o.get()[:, :, d if n else 0:] == 7.0).all()
    return oq.get()[:, :, :d], ok.get()[:, :, :d] if hk else None


def check_rotary(got, x, pos, sections, rot=None, dtype="f16", near=False, interleaved=False, spectra=False, theta=1e4, freq=None, **_):
    rot, of = rot or x.shape[2], pairs_of(sections, interleaved)
    n = len(of)
    # fractions of a turn in 128 bits: a frequency's turns per position as a whole number of 2^-128
    with localcontext() as how:
        how.prec = 80
        turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
        f = [Decimal(freq[i]) if freq is not None else Decimal(theta) ** (-Decimal(j) / Decimal(sections[a]) if spectra else -Decimal(i) / Decimal(n)) for i, (a, j) in enumerate(of)]
        f = np.array([int((v / turn * 2 ** 128).to_integral_value()) for v in f], dtype=object)
    angle = np.empty((x.shape[0], n))
    for p, (a, _) in enumerate(of):
        angle[:, p] = ((np.asarray(pos)[a].astype(object) * f[p] % (1 << 128)) >> 64).astype(np.float64) * (2 * np.pi / 2 ** 64)
    angle = torch.from_numpy(angle)[:, None]
    c, s = torch.cos(angle), torch.sin(angle)
    x = x.to(DT[dtype][0]).double()
    one, two = (slice(0, rot, 2), slice(1, rot, 2)) if near else (slice(0, n), slice(n, rot))
    a, b, want = x[:, :, one], x[:, :, two], x.clone()
    want[:, :, one], want[:, :, two] = a * c - b * s, b * c + a * s
    size = torch.zeros_like(x)
    size[:, :, one] = size[:, :, two] = a.abs() + b.abs()
    bound = DT[dtype][2] * want.abs() * 1.01 + TINY[dtype] + 8 * F32 * size
    assert torch.equal(got[:, :, rot:].double(), x[:, :, rot:])
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1, worst


ROTARY = [dict(rows=1, hq=1, hk=0, d=8, sections=[4]), dict(rows=3, hq=4, hk=2, d=64, sections=[16, 16]), dict(rows=130, hq=5, hk=1, d=128, sections=[16, 24, 24]),
          dict(rows=70, hq=2, hk=2, d=72, sections=[12, 12, 12]), dict(rows=33, hq=3, hk=3, d=80, rot=40, sections=[4, 16]), dict(rows=9, hq=2, hk=1, d=256, sections=[32, 32, 32, 32]),
          dict(rows=1000, hq=8, hk=8, d=32, rot=16, sections=[0, 8]), dict(rows=17, hq=1, hk=1, d=10, rot=6, sections=[1, 1, 1]), dict(rows=5, hq=300, hk=20, d=16, sections=[3, 5])]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("near,interleaved,spectra", [(False, False, False), (True, False, True), (False, True, False), (True, True, True)])
@pytest.mark.parametrize("case", ROTARY)
def test_rotary(gpu, case, dtype, near, interleaved, spectra):
    rows, d, how = case["rows"], case["d"], dict(sections=case["sections"], rot=case.get("rot"), dtype=dtype, near=near, interleaved=interleaved, spectra=spectra, theta=1e5)
    q, k = rand(d, rows, case["hq"], d) * 3, rand(d + 1, rows, case["hk"], d) if case["hk"] else None
    pos = np.random.default_rng(rows).integers(-50, 5000, (len(case["sections"]), rows))
    for layout in ("slices", "place", "heads", "odd"):
        a, b = rotary(q, k, pos, layout=layout, **how)
        check_rotary(a, q, pos, **how)
        if k is not None:
            check_rotary(b, k, pos, **how)


# pairs and copied channels that end inside a vector of 8 or 4: both, one alone, fewer than a vector
ODD = [dict(rows=400, hq=3, hk=2, d=26, sections=[13]), dict(rows=300, hq=2, hk=1, d=59, rot=58, sections=[15, 14]), dict(rows=200, hq=2, hk=2, d=67, rot=46, sections=[20, 3]),
       dict(rows=300, hq=1, hk=1, d=19, rot=16, sections=[8]), dict(rows=500, hq=1, hk=1, d=15, rot=10, sections=[5]), dict(rows=500, hq=2, hk=0, d=13, rot=8, sections=[4]),
       dict(rows=500, hq=2, hk=0, d=9, rot=4, sections=[1, 1]), dict(rows=100, hq=2, hk=1, d=255, rot=250, sections=[60, 65])]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("near", [False, True])
@pytest.mark.parametrize("case", ODD)
def test_rotary_odd_heads(gpu, case, near, dtype):
    """Every layout, and bit for bit the same in place."""
    rows, d, how = case["rows"], case["d"], dict(sections=case["sections"], rot=case.get("rot"), dtype=dtype, near=near)
    q, k = rand(d, rows, case["hq"], d) * 3, rand(d + 1, rows, case["hk"], d) if case["hk"] else None
    pos = np.random.default_rng(rows).integers(-50, 5000, (len(case["sections"]), rows))
    first = None
    for layout in ("slices", "place", "heads", "odd"):
        got = rotary(q, k, pos, layout=layout, **how)
        first = first or got
        for x, one, two in zip((q, k), first, got):
            if x is not None:
                check_rotary(two, x, pos, **how)
                assert torch.equal(one, two)


def test_rotary_far_positions_and_given_frequencies(gpu):
    """Both ends of the positions' range, and frequencies of any sign and size, whole turns and none among them."""
    q, k = rand(1, 8, 2, 64), rand(2, 8, 1, 64)
    pos = np.array([[0, -1, 1, 2 ** 31 - 1, -2 ** 31, 123456789, -987654321, 2 ** 30]])
    freq = [0.0, 1.0, -1.0, 2 * math.pi, 1e5, -3.7, 1e-12, 0.25] + list(np.geomspace(1e-6, 1e3, 24))
    for how in (dict(theta=1e4), dict(theta=5e5), dict(theta=1.0), dict(freq=freq)):
        a, b = rotary(q, k, pos, sections=[32], dtype="f32", **how)
        check_rotary(a, q, pos, sections=[32], dtype="f32", **how)
        check_rotary(b, k, pos, sections=[32], dtype="f32", **how)


def test_rotary_keeps_lengths_and_differences(gpu):
    """What it is for: products of turned rows go by the difference of their positions."""
    q, k = rand(3, 1, 1, 64).repeat(6, 1, 1), rand(4, 1, 1, 64).repeat(6, 1, 1)
    at = np.array([0, 5, 1000, 70000, 2 ** 20, 2 ** 30])
    a, _ = rotary(q, None, [at + 7, at + 3], sections=[20, 12], dtype="f32")
    b, _ = rotary(k, None, [at, at], sections=[20, 12], dtype="f32")
    z = (a.double() * b.double()).sum((1, 2))
    # 64 products of two outputs, each off by (8 + 1) 2^-24 of |a| + |b| at most
    assert (z - z[0]).abs().max() <= 64 * 2 * 9 * F32 * 2 * q.abs().max() * 2 * k.abs().max()


def test_rotary_special_values(gpu):
    """A NaN or infinity stays in its pair."""
    q = rand(5, 40, 2, 64)
    pos = np.arange(40)[None]
    clean, _ = rotary(q, None, pos, sections=[32])
    bad = q.clone()
    bad[7, 1, 3], bad[9, 0, 40] = float("nan"), float("inf")
    out, _ = rotary(bad, None, pos, sections=[32])
    touched = torch.zeros(q.shape, dtype=torch.bool)
    touched[7, 1, [3, 35]] = touched[9, 0, [8, 40]] = True
    assert torch.equal(out[~touched], clean[~touched]) and not torch.isfinite(out[touched]).any()


@pytest.mark.parametrize("rows,hq,hk,d,near", [(70001, 6, 2, 64, False), (20000, 33, 0, 40, False), (20000, 14, 2, 128, False), (20000, 14, 2, 128, True), (20000, 20, 1, 90, True)])
def test_rotary_many_rows(gpu, rows, hq, hk, d, near):
    """Enough rows for several heads a thread and, of whole lines, to pass the caches."""
    q, k = rand(6, rows, hq, d), rand(7, rows, hk, d) if hk else None
    how = dict(sections=[d // 4, d // 2 - d // 4], dtype="bf16", near=near)
    pos = np.stack([np.arange(rows) // 100, np.arange(rows) % 100])
    a, b = rotary(q, k, pos, **how)
    check_rotary(a, q, pos, **how)
    if hk:
        check_rotary(b, k, pos, **how)


# ------------------------------------------------------------------------------------ pages
class Pool:
    """A table, a list of free pages and both operators, beside the same in Python."""

    def __init__(self, batch, blocks, page, pages, capacity=None, seed=0):
        r = np.random.default_rng(seed)
        self.page, self.blocks, self.pages, self.batch, self.capacity = page, blocks, pages, batch, capacity or pages
        self.table, self.free, self.lost = [[-1] * blocks for _ in range(batch)], [int(v) for v in r.permutation(pages)], 0
        self.gpu_table, self.gpu_free = ints(self.table), ints((self.free + [-7] * self.capacity)[:self.capacity])
        self.state = ints([pages, 0])
        self.cache = V.KvCache(table=self.gpu_table.data_ptr(), pages=pages, page_tokens=page, kv_heads=1, head_dim=64, batch=batch, max_blocks=blocks)
        self.pool = V.KvPool(free=self.gpu_free.data_ptr(), state=self.state.data_ptr(), capacity=self.capacity)

    def count(self, tokens):
        return min(self.blocks, -(-max(tokens, 0) // self.page))

    def check(self):
        assert self.gpu_table.get().tolist() == self.table
        assert self.state.get().tolist() == [len(self.free), self.lost]
        assert self.gpu_free.get().tolist()[:len(self.free)] == self.free

    def reserve(self, lens, add, total, out=True, stream=None):
        cu, now = full((self.batch + 1,), -9, torch.int32), full((self.batch,), -9, torch.int32)
        pos, slot = full((max(total, 1),), -9, torch.int32), full((max(total, 1),), -9, torch.int64)
        dl, da = ints(lens), ints(add)
        sync()
        check(V.vkhip().vkhip_kv_reserve(R(self.cache), R(self.pool), dl.data_ptr(), da.data_ptr(), total, cu.data_ptr(), now.data_ptr() if out else None, pos.data_ptr() if out else None,
                                         slot.data_ptr() if out else None, stream), "kv_reserve")
        sync()
        most, want_cu, want_now, want_pos, want_slot = self.blocks * self.page, [0], [], [], []
        for b, (n, more) in enumerate(zip(lens, add)):
            n = min(max(n, 0), most)
            more = min(max(more, 0), total - want_cu[-1])
            for j in range(self.count(n), self.count(n + more)):
                self.table[b][j] = self.free.pop() if self.free else -1
                self.lost += self.table[b][j] < 0
            want_cu.append(want_cu[-1] + more)
            want_now.append(n + more)
            for t in range(n, n + more):
                name = self.table[b][t // self.page] if t < most else -1
                want_pos.append(t)
                want_slot.append(name * self.page + t % self.page if 0 <= name < self.pages else -1)
        assert cu.get().tolist() == want_cu
        behind = [-9] * (max(total, 1) - len(want_pos))  # rows that no sequence has stay as they were
        if out:
            assert now.get().tolist() == want_now and pos.get().tolist() == want_pos + behind and slot.get().tolist() == want_slot + behind
        self.check()
        return want_now

    def release(self, lens, keep):
        dl, dk = ints(lens), ints(keep)
        sync()
        check(V.vkhip().vkhip_kv_release(R(self.cache), R(self.pool), dl.data_ptr(), dk.data_ptr(), None), "kv_release")
        sync()
        given = []
        for b, (n, k) in enumerate(zip(lens, keep)):
            for j in range(self.count(min(k, self.blocks * self.page)), self.count(min(n, self.blocks * self.page))):
                given.append(self.table[b][j])
                self.table[b][j] = -1
        self.free = (self.free + [g for g in reversed(given) if 0 <= g < self.pages])[:self.capacity]
        self.check()


@pytest.mark.parametrize("page", [32, 64, 128, 256])
@pytest.mark.parametrize("batch", [1, 2, 63, 1024, 1025, 2500])
def test_pages_over_steps(gpu, page, batch):
    """Prompts, single tokens, drafts taken back, sequences that end and others that begin in their place."""
    r = np.random.default_rng(page + batch)
    p = Pool(batch, 9, page, batch * 5 + 3, seed=page)
    lens = [0] * batch
    for step in range(6):
        add = [int(v) for v in (r.integers(0, 2 * page, batch) if step % 3 == 0 else r.integers(0, 2, batch) if step % 3 == 1 else r.integers(0, 6, batch))]
        add = [min(a, 8 * page - n) for a, n in zip(add, lens)]
        now = p.reserve(lens, add, sum(add))
        keep = [0 if r.random() < 0.2 else max(0, n - int(r.integers(0, 4))) for n in now]
        p.release(now, keep)
        lens = keep
    everything = [n for n in lens]
    p.release(everything, [0] * batch)
    assert sorted(p.free) == list(range(batch * 5 + 3)) or p.lost


def test_pages_back_in_order(gpu):
    """What goes back is what the same reserve takes again."""
    p = Pool(7, 6, 64, 60, seed=3)
    lens, add = [0, 64, 65, 1, 0, 200, 63], [130, 1, 0, 63, 64, 100, 2]
    start = p.reserve([0] * 7, lens, sum(lens))
    now = p.reserve(start, add, sum(add))
    before = [list(t) for t in p.table]
    p.release(now, start)
    p.reserve(start, add, sum(add))
    assert p.table == before


def test_pages_run_out(gpu):
    """Blocks without a page in the list are blocks without memory, counted; the list is never read past its start."""
    p = Pool(5, 8, 32, 11, seed=4)
    now = p.reserve([0] * 5, [70, 70, 70, 70, 70], 350)
    assert p.lost == 4 and p.table[4] == [-1] * 8
    now = p.reserve(now, [60] * 5, 300)
    p.release(now, [0, 64, 0, 0, 0])
    assert len(p.free) == 9
    empty = Pool(3, 4, 32, 0, capacity=2)
    empty.reserve([0, 0, 0], [1, 40, 0], 41)


def test_pages_lists_and_lengths_out_of_range(gpu):
    """Lengths, sums and names that make no sense stay within the arrays."""
    p = Pool(4, 3, 32, 20, seed=5)
    p.reserve([-5, 96, 1 << 30, 0], [3, 1, 2, -4], 6)  # nothing of a full table or a negative count
    p.reserve([0, 0, 0, 0], [50, 1 << 30, (1 << 31) - 1, 10], 60)  # cut to the rows there are
    p.reserve([90, 0, 0, 95], [20, 0, 0, 2], 22)  # tokens past the table have a position and no slot
    names = p.gpu_table.get()
    names[0, 0], names[1, 1] = 77, -3
    p.gpu_table.put(names)
    p.table = names.tolist()
    p.release([96, 96, -1, 500], [0, 0, 0, 0])
    small = Pool(2, 4, 32, 6, capacity=6, seed=6)
    now = small.reserve([0, 0], [100, 60], 160)
    small.capacity, small.pool.capacity = 3, 3  # no room for all that comes back
    small.release(now, [0, 0])
    assert len(small.free) == 3


@pytest.mark.parametrize("batch,most", [(3, 9000), (64, 500), (300, 90)])
def test_pages_of_prompts(gpu, batch, most):
    """More rows than one workgroup writes along with the table."""
    r = np.random.default_rng(batch)
    lens, add = ([int(v) for v in r.integers(0, n, batch)] for n in (300, most))
    p = Pool(batch, 300 // 64 + most // 64 + 2, 64, batch * (most // 64 + 7), seed=1)
    p.reserve([0] * batch, lens, sum(lens) + 5)
    p.reserve(lens, add, sum(add) + 5)
    p.reserve(lens, add, sum(add) // 2)
    p.reserve(lens, add, sum(add), out=False)


# ------------------------------------------------------------------------------------ shared prefixes
def shared_cache(sizes, prefixes, tails, page, heads, d, outside=0, seed=0, blocks=None):
    """Groups of sequences whose first blocks are the first one's; `outside` sequences in front of them and behind share
    nothing and have a tail alone. Returns the cache, lengths, cu, prefixes."""
    of = [-1] * outside + [g for g, n in enumerate(sizes) for _ in range(n)] + [-1] * outside
    pre = [0 if g < 0 else prefixes[g] for g in of]
    lens = [p + t for p, t in zip(pre, tails)]
    c = T.Cache(len(of), blocks or max(1, -(-max(lens) // page)), page, heads, d, seed)
    cu = [outside + int(x) for x in np.cumsum([0] + list(sizes))]
    lead = [b in [cu[g] for g, n in enumerate(sizes) if n] and of[b] >= 0 for b in range(len(of))]
    for b in range(len(of)):
        if of[b] >= 0:
            c.table[b, :pre[b] // page] = c.table[cu[of[b]], :pre[b] // page]
    c.gpu_table.put(c.table)

    def rows(n, salt):
        return rand(seed + salt, n, heads, d) * (1 + torch.arange(n)[:, None, None] // 40 % 5)
    first = [p if is_lead else 0 for p, is_lead in zip(pre, lead)]
    if sum(first):
        c.append(rows(sum(first), 1), rows(sum(first), 2), first, [0] * len(of), "f16")
    if sum(tails):
        c.append(rows(sum(tails), 3), rows(sum(tails), 4), list(tails), pre, "f16")
    return c, lens, cu


def widen(c, rows, tiles):
    """A table so wide that, as far as the host knows, prefixes of that many tokens times `rows` rows a sequence are worth tiles
    of 128 or 256 rows (None: as it is)."""
    if tiles:
        work = 3 << 24 if c.d <= 64 else 3 << 22 if tiles == 128 else 1 << 24
        c.blocks = max(c.blocks, work // (c.heads * c.batch * rows * c.page) + 1)
        c.table = torch.cat([c.table, torch.full((c.batch, c.blocks - c.table.shape[1]), -1, dtype=torch.int32)], 1).contiguous()
        c.gpu_table = Dev(c.table)


def shared_attention(c, q, lens, cu, prefixes, dtype, scale, max_len=0, max_tokens=0, max_tail=0, stream=None, o_pad=0):
    """q [batch, t, heads, d]"""
    lib, (dt, code, _) = V.vkhip(), DT[dtype]
    dq = Dev(q.to(dt))
    b, t, hq, d = q.shape
    out = full((b, t, hq, d + o_pad), 7.0, dt)
    desc = V.KvAttentionDesc(q_heads=hq, q_tokens=t, dtype=code, max_len=max_len, scale=scale, q_row=hq * d, q_head=d, o_row=hq * (d + o_pad), o_head=d + o_pad)
    cd, n, dc, dp = c.desc(), ints(lens), ints(cu), ints(list(prefixes) or [0])
    p = V.KvPrefix(cu=dc.data_ptr(), tokens=dp.data_ptr(), groups=len(cu) - 1, max_tokens=max_tokens, max_tail=max_tail)
    ws = workspace(lib.vkhip_kv_attention_shared_workspace_bytes(R(desc), R(cd), R(p)))
    sync()
    check(lib.vkhip_kv_attention_shared(R(desc), R(cd), R(p), dq.data_ptr(), n.data_ptr(), out.data_ptr(), ws.data_ptr(), stream), "kv_attention_shared")
    sync()
    out = out.get()
    assert (out[..., d:] == 7.0).all()
    return out[..., :d].double()


def both_checks(c, q, lens, cu, prefixes, dtype, scale, **how):
    out = shared_attention(c, q, lens, cu, prefixes, dtype, scale, o_pad=8, **how)
    T.check_kv_attention(out, c, q, lens, dtype, scale)


GROUPS = [([1], [64]), ([4], [256]), ([2, 3], [0, 128]), ([5, 0, 1, 40], [512, 256, 0, 1024]), ([70], [768]), ([3, 3, 3], [256, 256, 256])]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("page,t", [(32, 1), (64, 1), (64, 3), (256, 2)])
@pytest.mark.parametrize("sizes,prefixes", GROUPS)
@pytest.mark.parametrize("hq,hkv,d", [(4, 4, 64), (8, 2, 128), (7, 1, 72)])
def test_shared(gpu, dtype, page, t, sizes, prefixes, hq, hkv, d):
    prefixes = [p // page * page for p in prefixes]
    r = np.random.default_rng(sum(sizes))
    tails = [int(v) for v in r.integers(t, 150, sum(sizes) + 2)]
    c, lens, cu = shared_cache(sizes, prefixes, tails, page, hkv, d, outside=1, seed=d + t)
    q = rand(9, len(lens), t, hq, d).to(DT[dtype][0]).float()
    both_checks(c, q, lens, cu, prefixes, dtype, d ** -0.5)


@pytest.mark.parametrize("sizes,hq,hkv,t", [([130], 8, 2, 1), ([9, 60], 16, 2, 3), ([33], 32, 4, 1), ([200, 1], 4, 4, 1), ([17], 64, 1, 2)])
@pytest.mark.parametrize("page,prefixes", [(32, [1056, 2016]), (64, [2048, 64]), (128, [128, 3968])])
def test_shared_many_rows(gpu, sizes, hq, hkv, t, page, prefixes):
    """Groups whose rows fill several tiles of 128."""
    tails = [t + i % 50 for i in range(sum(sizes))]
    prefixes = prefixes[:len(sizes)]
    for d, dtype in ((128, "f16"), (64, "bf16"), (88, "bf16")):
        c, lens, cu = shared_cache(sizes, prefixes, tails, page, hkv, d, seed=t)
        q = rand(10, len(lens), t, hq, d).to(DT[dtype][0]).float()
        for tiles in (None, 128, 256) if d == 128 else (256,):
            widen(c, hq // hkv * t, tiles)
            both_checks(c, q, lens, cu, prefixes, dtype, d ** -0.5, max_tokens=0 if tiles else max(prefixes), max_tail=max(tails))


@pytest.mark.parametrize("many,tiles,page,d", [(5, None, 64, 128), (60, None, 64, 128), (60, 256, 64, 128), (9, 128, 64, 128), (60, 128, 64, 64), (60, 256, 32, 128), (60, 128, 32, 72)])
def test_shared_lengths_inside_the_prefix(gpu, many, tiles, page, d):
    """Sequences that have not reached their prefix's end, the first one's table naming it: they see what their length
    lets them. A length of nothing gives zeros, more query tokens than tokens give rows that see nothing."""
    heads, t = 2, 4
    c, lens, cu = shared_cache([many], [512], [t] * many, page, heads, d)
    for b in range(many):
        c.table[b] = c.table[0]  # all are the first's prefix
    c.gpu_table.put(c.table)
    widen(c, t * 4, tiles)
    lens = [[512, 511, 0, 1, 3, 64, 65, 300, 449, 2][b % 10] for b in range(many)]
    q = rand(11, many, t, 8, d).half().float()
    out = shared_attention(c, q, lens, cu, [512], "f16", 0.09)
    T.check_kv_attention(out, c, q, lens, "f16", 0.09)
    assert (out[2] == 0).all() and (out[3][:3] == 0).all()


@pytest.mark.parametrize("many,tiles,d", [(4, None, 64), (64, None, 64), (64, 128, 64), (64, 256, 128), (20, 128, 128)])
def test_shared_spoiled_and_missing_pages(gpu, many, tiles, d):
    """A prefix page of NaN scale reaches the queries that see it and no other; one without memory is seen by none; the
    tails' and the other group's pages stay their own."""
    page, heads = 64, 1
    c, lens, cu = shared_cache([many, many], [256, 192], [5] * (2 * many), page, heads, d, seed=3)
    widen(c, 4, tiles)
    q = rand(12, 2 * many, 1, 4, d).half().float()
    clean = shared_attention(c, q, lens, cu, [256, 192], "f16", 0.125)
    for scales in (c.ks, c.vs):
        spoiled, was = scales.get(), scales.get()
        spoiled[int(c.table[0, 3])] = float("nan")  # tokens 192 .. 255 of the first group
        scales.put(spoiled)
        short = [200 if b == 1 else 150 if b == 2 else n for b, n in enumerate(lens)]
        out = shared_attention(c, q, short, cu, [256, 192], "f16", 0.125)
        assert torch.equal(out[many:], clean[many:]) and torch.isfinite(out[2]).all()
        assert torch.isnan(out[[0, 1, 3]]).all()
        scales.put(was)
    names = c.table.clone()
    names[0, 1], names[many, 2], names[many + 1, 3] = -1, c.pages + 5, 1 << 30
    c.gpu_table.put(names)
    out = shared_attention(c, q, lens, cu, [256, 192], "f16", 0.125)
    for b, gone in [(b, range(64, 128)) for b in range(many)] + [(many, range(128, 192)), (many + 1, range(128, 197))]:
        (kq, ks), (vq, vs) = c.bytes_of(b, lens[b])
        keep = torch.ones(lens[b], dtype=torch.bool)
        keep[list(gone)] = False
        k, v = (kq.double() * ks.double()[:, :, None])[keep], (vq.double() * vs.double()[:, :, None])[keep]
        T.check_attention(out[b], q[b].double(), k, v, [1], [int(keep.sum())], True, "f16", 0.125)


@pytest.mark.parametrize("sizes,hq,tiles", [([3, 20], 4, None), ([20, 30], 16, 128), ([20, 30], 16, 256)])
def test_shared_hints_and_odd_prefixes(gpu, sizes, hq, tiles):
    """Prefixes are whole pages; a smaller max_tokens leaves the rest to the tails, a smaller max_tail costs time alone,
    max_len cuts sequences; a wide table changes nothing."""
    page, heads, d = 64, 2, 128
    many = sum(sizes)
    c, lens, cu = shared_cache(sizes, [640, 192], [10 + b % 23 for b in range(many)], page, heads, d, seed=6, blocks=40)
    q = rand(13, many, 1, hq, d).half().float()
    widen(c, hq // heads, tiles)
    for how in (dict(), dict(max_tokens=640, max_tail=32), dict(max_tokens=300), dict(max_tokens=64), dict(max_tokens=63), dict(max_tail=1), dict(max_len=700), dict(max_tokens=1 << 20)):
        for given in ([640, 192], [703, 193], [641, 255]):
            both_checks(c, q, lens, cu, given, "f16", 0.09, **how)
    out = shared_attention(c, q, lens, cu, [640, 192], "f16", 0.09, max_len=100)
    T.check_kv_attention(out, c, q, [min(100, n) for n in lens], "f16", 0.09)
    both_checks(c, q, lens, cu, [0, -5], "f16", 0.09)
    both_checks(c, q, lens, [0], [], "f16", 0.09)  # no groups


def test_shared_groups_out_of_range(gpu):
    """Ranges and prefixes that make no sense stay within the arrays, and sequences in no group are right."""
    c, lens, cu = shared_cache([4], [128], [20] * 4, 64, 1, 64, seed=7)
    q = rand(14, 4, 1, 2, 64).half().float()
    wide, many, wcu = shared_cache([70], [128], [20] * 70, 64, 1, 64, seed=7)  # the same in wide tiles
    widen(wide, 2, 128)
    wq = rand(14, 70, 1, 2, 64).half().float()
    for given in ([0, 1 << 30], [-7, 70], [5, 66]):
        for prefix in (128, 0, -64):
            both_checks(wide, wq, many, given, [prefix], "f16", 0.125)
    both_checks(c, q, lens, [0, 1 << 30], [128], "f16", 0.125)
    both_checks(c, q, lens, [-7, 4], [128], "f16", 0.125)
    both_checks(c, q, lens, [2, 2, 2], [128, 1 << 30], "f16", 0.125)
    out = shared_attention(c, q, lens, [0, 4], [-64], "f16", 0.125)
    T.check_kv_attention(out, c, q, lens, "f16", 0.125)


def test_shared_many_groups(gpu):
    """More groups than a wave has lanes, empty ones among them."""
    r = np.random.default_rng(8)
    sizes = [int(v) for v in r.integers(0, 4, 150)]
    prefixes = [int(v) * 64 for v in r.integers(0, 4, 150)]
    c, lens, cu = shared_cache(sizes, prefixes, [int(v) for v in r.integers(1, 80, sum(sizes) + 2)], 64, 1, 64, outside=1, seed=8)
    q = rand(15, len(lens), 1, 4, 64).half().float()
    both_checks(c, q, lens, cu, prefixes, "f16", 0.125)


@pytest.mark.parametrize("many,tiles,d", [(2, None, 64), (40, None, 64), (40, 128, 64), (130, 128, 64), (60, 256, 128)])
def test_shared_large_scores(gpu, many, tiles, d):
    """bf16 queries beyond fp16's range, scores in the thousands, keys that grow along the prefix: maxima that move late."""
    page, heads = 64, 2
    c, lens, cu = shared_cache([many], [1024], [30] * many, page, heads, d, seed=9)
    ks = c.ks.get()
    ks[c.table[0, :16].long()] *= torch.linspace(0.1, 8, 16)[:, None]
    c.ks.put(ks)
    widen(c, 4, tiles)
    q = (rand(16, many, 1, 8, d) * torch.tensor([1e-6, 1.0, 1e5, 1e9] * 2)[None, None, :, None]).bfloat16().float()
    for scale in (1e-9, 1e-5, 1.0):
        both_checks(c, q, lens, cu, [1024], "bf16", scale)


@pytest.mark.parametrize("many,tiles,page,d", [(2, None, 64, 64), (40, None, 64, 64), (40, 128, 64, 64), (60, 256, 64, 128), (40, 128, 32, 64), (60, 256, 32, 128), (20, 128, 32, 128)])
def test_shared_value_scales_far_apart(gpu, many, tiles, page, d):
    """Pages of values many powers of two apart, and one of zeros: a small page that owns the weights keeps its digits
    beside a large one that has none."""
    heads = 1
    c, lens, cu = shared_cache([many], [512], [3] * many, page, heads, d, seed=10)
    widen(c, 4, tiles)
    vs, ks = c.vs.get(), c.ks.get()
    for i, f in enumerate([1.0, 2.0 ** -30, 2.0 ** 20, 0.0, 2.0 ** -60, 1.0, 2.0 ** 10, 1.0]):
        vs[int(c.table[0, i])] *= f
    c.vs.put(vs)
    q = rand(17, many, 1, 4, d).half().float()
    for own in (1, 4, 6):  # the page whose keys are large: its best key takes nearly all
        now = ks.clone()
        now[int(c.table[0, own])] *= 60
        c.ks.put(now)
        out = shared_attention(c, q, lens, cu, [512], "f16", 1.0)
        for b in (0, many - 1):
            (kq, ksc), (vq, vsc) = c.bytes_of(b, lens[b])
            k, v = kq.double() * ksc.double()[:, :, None], vq.double() * vsc.double()[:, :, None]
            see = torch.ones(1, lens[b], dtype=torch.bool)
            for h in range(4):
                want, pv, qk = T.attention64(q[b, :, h].double(), k[:, 0], v[:, 0], see, 1.0)
                # a weight is rounded once, and what lies under 2^-38 of a row's largest may be lost
                p = torch.softmax(q[b, :, h].double() @ k[:, 0].T, 1)
                e = (d + 16) * F32 * qk + 2.0 ** -20
                bound = 2.0 ** -11 * want.abs() * 1.01 + TINY["f16"] + (2.0 ** -11 * 1.02 + 2 * e) * pv + p.clamp(max=2.0 ** -38) @ v[:, 0].abs()
                assert ((out[b, :, h] - want).abs() / bound).max().item() <= 1, (own, b, h)


@pytest.mark.parametrize("many,tiles,page,d", [(5, None, 64, 64), (40, 128, 64, 64), (60, 256, 64, 128), (40, 128, 32, 64)])
def test_shared_pages_of_zeros(gpu, many, tiles, page, d):
    """Pages whose keys, values or both are zeros: scores of nothing that still take their weight, and a prefix of such alone."""
    c, lens, cu = shared_cache([many], [512], [3] * many, page, 1, d, seed=18)
    widen(c, 4, tiles)
    vs, ks = c.vs.get(), c.ks.get()
    q = rand(19, many, 1, 4, d).half().float()
    for keys, values in (([1, 2, 7], [2, 5]), (range(512 // page), []), (range(512 // page), range(512 // page))):
        a, b = ks.clone(), vs.clone()
        a[[int(c.table[0, i]) for i in keys]] = 0.0
        b[[int(c.table[0, i]) for i in values]] = 0.0
        c.ks.put(a)
        c.vs.put(b)
        both_checks(c, q, lens, cu, [512], "f16", 0.125)


def test_shared_long_prefix(gpu):
    """Offsets past 2^31 bytes: the prefix's pages lie at the end of a large pool."""
    page, heads, d = 64, 8, 128
    pages, blocks, many = (1 << 31) // (heads * page * d) + 700, 520, 3
    c = T.Cache.__new__(T.Cache)
    c.page, c.heads, c.d, c.dp, c.batch, c.blocks, c.pages = page, heads, d, 128, many, blocks, pages
    c.table = (pages - 1 - torch.arange(blocks * many)).view(many, blocks).int()
    c.table[1:, :512] = c.table[0, :512]
    c.gpu_table = Dev(c.table)
    c.k, c.v = Dev.zeros((pages, heads, page, d), torch.int8), Dev.zeros((pages, heads, d, page), torch.int8)
    c.ks, c.vs = Dev.zeros((pages, heads), torch.float32), Dev.zeros((pages, heads), torch.float32)
    k, v = rand(1, 32768, heads, d), rand(2, 32768, heads, d)
    c.append(k, v, [32768, 0, 0], [0, 0, 0], "f16")
    c.append(k[:90], v[:90], [30, 50, 10], [32768] * 3, "f16")
    lens = [32798, 32818, 32778]
    q = rand(3, many, 1, 16, d).half().float()
    both_checks(c, q, lens, [0, 3], [32768], "f16", 0.09, max_tail=50)


# ------------------------------------------------------------------------------------ norms around a block
def residual_norm(x, r, dtype="f16", post="rms", pre="rms", alpha=1.0, post_w=None, post_b=None, pre_w=None, pre_b=None, gate=None, scale=None, shift=None, mod=None, mod_rows=0,
                  post_eps=1e-5, pre_eps=1e-6, pad=0, place=None, want=("h", "y"), stream=None):
    """x, r [rows, dim] or None; gate, scale, shift [mods, dim] or None. place: h over "x" or "r", y over the other."""
    lib, (dt, code, _) = V.vkhip(), DT[dtype]
    rows, dim = (x if x is not None else r).shape

    def padded(t):
        if t is None:
            return None
        return Dev(torch.cat([t, torch.full((t.shape[0], pad), 5.0)], 1).to(dt))
    dx, dr = padded(x), padded(r)
    vec = [None if t is None else padded(t) for t in (gate, scale, shift)]
    mods = next((t.shape[0] for t in (gate, scale, shift) if t is not None), 0)
    h, y = (full((rows, dim + pad), 7.0, dt) for _ in range(2))
    if place:
        h, y = (dx, dr) if place == "x" else (dr, dx)
    ws = [None if t is None else Dev(t.float()) for t in (post_w, post_b, pre_w, pre_b)]
    dm = None if mod is None else ints(mod)
    d = V.ResidualNormDesc(rows=rows, dim=dim, dtype=code, post=V.NORM[post], pre=V.NORM[pre], mods=mods, mod_rows=mod_rows, alpha=alpha, post_eps=post_eps, pre_eps=pre_eps, x_row=dim + pad,
                           r_row=dim + pad, h_row=dim + pad, y_row=dim + pad, mod_row=dim + pad)

    def ptr(t):
        return None if t is None else t.data_ptr()
    sync()
    check(lib.vkhip_residual_norm(R(d), ptr(dx), ptr(dr), ptr(ws[0]), ptr(ws[1]), ptr(vec[0]), ptr(ws[2]), ptr(ws[3]), ptr(vec[1]), ptr(vec[2]), ptr(dm), ptr(h) if "h" in want else None,
                                  ptr(y) if "y" in want else None, stream), "residual_norm")
    sync()
    beside = 5.0 if place else 7.0
    outs = [t.get() for t in (h, y)]
    for t, name in zip(outs, "hy"):
        assert (t[:, dim:] == beside).all() and (name in want or (t == 7.0).all())
    return [t[:, :dim].double() for t in outs]


def norm64(z, dz, kind, w, b, eps):
    """The norm of z and how far it may be off, given how far z is."""
    if kind == "none":
        return z, dz
    w = torch.ones(z.shape[1], dtype=torch.float64) if w is None else w.double()
    b = torch.zeros(z.shape[1], dtype=torch.float64) if b is None else b.double()
    mean = z.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(z[:, :1])
    rms = ((z - mean).square().mean(1, keepdim=True) + eps).sqrt()
    n, dr = (z - mean) / rms, dz.square().mean(1, keepdim=True).sqrt()
    off = 64 * F32 * (n.abs() * w.abs() + (mean.abs() + z.abs().mean(1, keepdim=True)) / rms * w.abs() + w.abs() + b.abs())
    return n * w + b, off + (dz + dr * (1 + n.abs())) / rms * w.abs()


def check_norm(got, x, r, dtype="f16", post="rms", pre="rms", alpha=1.0, post_w=None, post_b=None, pre_w=None, pre_b=None, gate=None, scale=None, shift=None, mod=None, mod_rows=0,
               post_eps=1e-5, pre_eps=1e-6, want=("h", "y"), **_):
    dt, _, u = DT[dtype]
    rows = (x if x is not None else r).shape[0]
    # without an index and a number of rows there is one vector for all
    at = torch.tensor(mod, dtype=torch.long) if mod is not None else torch.arange(rows) // mod_rows if mod_rows else torch.zeros(rows, dtype=torch.long)

    def vector(t):
        return t.to(dt).double()[at.clamp(0, t.shape[0] - 1)]
    alpha = float(np.float32(alpha))
    h, dh = torch.zeros((1, 1), dtype=torch.float64), 0
    if x is not None:
        f, df = norm64(x.to(dt).double(), torch.zeros_like(x, dtype=torch.float64), post, post_w, post_b, float(np.float32(post_eps)))
        g = alpha * (vector(gate) if gate is not None else 1.0)
        h, dh = f * g, (df + 3 * F32 * f.abs()) * abs(g)
    if r is not None:
        h = h + r.to(dt).double()
    dh = dh + F32 * h.abs()
    y, dy = norm64(h, dh, pre, pre_w, pre_b, float(np.float32(pre_eps)))
    if scale is not None:
        y, dy = y * (1 + vector(scale)), (dy + 2 * F32 * y.abs()) * (1 + vector(scale).abs())
    if shift is not None:
        y, dy = y + vector(shift), dy + F32 * (y.abs() + vector(shift).abs())
    for name, t, off, out in (("h", h, dh, got[0]), ("y", y, dy, got[1])):
        if name in want:
            worst = ((out - t).abs() / (u * t.abs() * 1.01 + off * 1.01 + TINY[dtype])).max().item()
            assert worst <= 1, (name, worst)


NORM_SIZES = [(1, 1), (3, 7), (2, 16), (5, 100), (70, 64), (9, 512), (4, 513), (3, 1100), (2, 2048), (3, 2056), (2, 4096), (1, 5001), (2, 8192), (1, 8200), (2, 16384), (1, 20001), (1, 32768)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
def test_residual_norm(gpu, rows, dim, dtype):
    """Every pair of norms over the sizes: with and without weights, vectors by an index, by rows, or none."""
    x, r = rand(dim, rows, dim) * 2 + 0.5, rand(dim + 1, rows, dim) * 5 - 1
    w = [rand(i, dim) * 0.3 + 1 for i in range(4)]
    vec = [rand(10 + i, 3, dim) for i in range(3)]
    mod = [(i * 2) % 5 - 1 for i in range(rows)]  # -1 and 3 are clamped
    for i, (post, pre) in enumerate([(a, b) for a in ("none", "rms", "layer") for b in ("none", "rms", "layer")]):
        how = dict(dtype=dtype, post=post, pre=pre, alpha=[1.0, 0.3, -1.5][i % 3])
        if i % 2:
            how.update(post_w=w[0], pre_w=w[2], pre_b=w[3])
        if i % 3 == 1:
            how.update(gate=vec[0], scale=vec[1], shift=vec[2], mod=mod)
        if i % 3 == 2:
            how.update(gate=vec[0], post_b=w[1], mod_rows=-(-rows // 3))
        check_norm(residual_norm(x, r, pad=8 if dim % 8 == 0 else 4 if dim % 4 == 0 else 1, **how), x, r, **how)


def test_residual_norm_parts_alone(gpu):
    """No block, no residual, one output, one vector for all rows; in place both ways."""
    x, r, g = rand(1, 40, 96), rand(2, 40, 96), rand(3, 1, 96)
    for how in (dict(x=None, r=r), dict(x=x, r=None), dict(x=x, r=r, want="h"), dict(x=x, r=r, want="y"), dict(x=None, r=r, want="y", pre="layer"), dict(x=x, r=r, gate=g), dict(x=x, r=r, scale=g),
                dict(x=x, r=r, shift=g), dict(x=None, r=r, gate=g, shift=g, want="y"), dict(x=x, r=r, place="x", gate=g), dict(x=x, r=r, place="r", pad=8)):
        args = dict(how)
        check_norm(residual_norm(args.pop("x"), args.pop("r"), **args), **how)


def test_residual_norm_far_from_zero_and_no_variance(gpu):
    """A mean of 2000 deviations, rows of one value, rows of zeros with no eps's help but eps."""
    x = (rand(5, 6, 900) + 2000).float()
    how = dict(dtype="f32", post="layer", pre="layer")
    check_norm(residual_norm(x, None, **how), x, None, **how)
    flat = torch.full((3, 77), 3.0)
    assert (residual_norm(None, flat, dtype="f32", pre="layer")[1] == 0).all()
    assert (residual_norm(flat * 0, flat * 0, dtype="f32", post="layer", pre="rms")[1] == 0).all()


def test_residual_norm_spoiled_row(gpu):
    """NaN and infinities stay in their row."""
    x, r = rand(6, 9, 300), rand(7, 9, 300)
    clean = residual_norm(x, r)
    bad = x.clone()
    bad[4, 7], bad[6, 0] = float("nan"), float("inf")
    out = residual_norm(bad, r)
    for a, b in zip(clean, out):
        keep = [i for i in range(9) if i not in (4, 6)]
        assert torch.equal(a[keep], b[keep]) and torch.isnan(b[4]).all()


@pytest.mark.parametrize("dim,dtype", [(5, "bf16"), (8, "bf16"), (88, "bf16"), (200, "f16"), (2047, "f16"), (2048, "bf16")])
def test_residual_norm_many_rows(gpu, dim, dtype):
    """More rows than run at once: every one is written, as its own."""
    rows = 20011
    x, r = rand(8, 7, dim).repeat(rows // 7 + 1, 1)[:rows], rand(9, 11, dim).repeat(rows // 11 + 1, 1)[:rows]
    h, y = residual_norm(x, r, dtype=dtype, pre="layer")
    check_norm([h[:77], y[:77]], x[:77], r[:77], dtype=dtype, pre="layer")
    at = torch.arange(rows) % 77
    assert torch.equal(h, h[at]) and torch.equal(y, y[at])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("rows,dim", [(700, 9), (333, 67), (333, 131), (301, 259), (300, 515), (300, 1029), (300, 1541), (200, 2302), (200, 3100), (100, 5003), (60, 7001), (40, 8193), (20, 16389), (9, 24581)])
def test_residual_norm_odd_rows_in_place(gpu, rows, dim, dtype):
    """Rows whose last vector begins inside the one before, in place: bit for bit as elsewhere, with and without a norm between loads and stores."""
    x, r, g = rand(1, rows, dim), rand(2, rows, dim), rand(3, 1, dim)
    for how in (dict(post="none", pre="none", gate=g), dict(post="layer", pre="layer")):
        apart = residual_norm(x, r, dtype=dtype, **how)
        check_norm(apart, x, r, dtype=dtype, **how)
        for place in ("x", "r"):
            for one, two in zip(apart, residual_norm(x, r, dtype=dtype, place=place, pad=1, **how)):
                assert torch.equal(one, two)


# ------------------------------------------------------------------------------------ together
def test_step_on_a_stream_of_its_own_and_as_a_graph(gpu):
    """Two steps of several requests behind a shared prefix as they would be used: norm, pages, positions, rows into the
    cache, attention, norm with the residual; eager, and as a graph replayed with the program's own work between."""
    lib = V.vkhip()
    s, g = ctypes.c_void_p(), ctypes.c_void_p()
    check(lib.vkhip_stream_create(ctypes.byref(s)))
    page, hkv, hq, d, n, many, pre = 64, 2, 4, 64, 5, 2, 128
    dim = hq * d
    c, lens, cu = shared_cache([n], [pre], [63, 1, 62, 100, 126], page, hkv, d, seed=11, blocks=8)
    used = {int(v) for b in range(n) for v in c.table[b, :-(-lens[b] // page)]}
    free = [i for i in range(c.pages) if i not in used]
    names = c.table.clone()
    for b in range(n):
        names[b, -(-lens[b] // page):] = -1
    rows = n * many
    x, r, h, y, att = (full((rows, dim), 0.0, torch.float16) for _ in range(5))
    q, k = full((rows, dim), 0.0, torch.float16), full((rows, hkv * d), 0.0, torch.float16)
    v = Dev(rand(3, rows, hkv * d).half())
    was, add, now, dcu, pos, slot = ints(lens), ints([many] * n), ints([0] * n), ints([0] * (n + 1)), ints([0] * rows), Dev.zeros((rows,), torch.int64)
    dfree, state, dc, dp = ints(free), ints([len(free), 0]), ints(cu), ints([pre])
    pool, cd = V.KvPool(free=dfree.data_ptr(), state=state.data_ptr(), capacity=len(free)), c.desc()
    nd = V.ResidualNormDesc(rows=rows, dim=dim, dtype=0, post=1, pre=1, alpha=1.0, post_eps=1e-5, pre_eps=1e-5, x_row=dim, r_row=dim, h_row=dim, y_row=dim)
    rd = V.RotaryDesc(rows=rows, q_heads=hq, k_heads=hkv, head_dim=d, rotary_dim=d, dtype=0, axes=1, sections=(32, 0, 0, 0), theta=1e4, q_row=dim, q_head=d, k_row=dim, k_head=d, qo_row=dim,
                      qo_head=d, ko_row=hkv * d, ko_head=d)
    kr = V.KvRows(dtype=0, total=rows, k_row=hkv * d, k_head=d, v_row=hkv * d, v_head=d)
    ad = V.KvAttentionDesc(q_heads=hq, q_tokens=many, dtype=0, max_len=page * 8, scale=0.125, q_row=dim, q_head=d, o_row=dim, o_head=d)
    pf = V.KvPrefix(cu=dc.data_ptr(), tokens=dp.data_ptr(), groups=1, max_tokens=pre, max_tail=200)
    ws = workspace(lib.vkhip_kv_attention_shared_workspace_bytes(R(ad), R(cd), R(pf)))

    def chain():
        check(lib.vkhip_residual_norm(R(nd), None, x.data_ptr(), None, None, None, None, None, None, None, None, None, y.data_ptr(), s))
        check(lib.vkhip_kv_reserve(R(cd), R(pool), was.data_ptr(), add.data_ptr(), rows, dcu.data_ptr(), now.data_ptr(), pos.data_ptr(), slot.data_ptr(), s))
        check(lib.vkhip_rotary(R(rd), pos.data_ptr(), None, y.data_ptr(), y.data_ptr(), q.data_ptr(), k.data_ptr(), s))
        check(lib.vkhip_kv_append(R(cd), R(kr), k.data_ptr(), v.data_ptr(), dcu.data_ptr(), was.data_ptr(), s))
        check(lib.vkhip_kv_attention_shared(R(ad), R(cd), R(pf), q.data_ptr(), now.data_ptr(), att.data_ptr(), ws.data_ptr(), s))
        check(lib.vkhip_residual_norm(R(nd), att.data_ptr(), x.data_ptr(), None, None, None, None, None, None, None, None, h.data_ptr(), r.data_ptr(), s))

    def start():
        c.gpu_table.put(names)
        dfree.put(torch.tensor(free, dtype=torch.int32))
        state.put(torch.tensor([len(free), 0], dtype=torch.int32))
        for t in (h, r, att, q, k, y):
            t.put(torch.full(t.shape, 9.0, dtype=t.dtype))
        sync()
    start()
    kept = [c.k.get(), c.v.get(), c.ks.get(), c.vs.get()]
    check(lib.vkhip_graph_begin(s))
    chain()
    check(lib.vkhip_graph_end(s, ctypes.byref(g)))
    for i in range(4):
        x.put(rand(i, rows, dim).half())
        got = []
        for how in ("eager", "graph"):
            start()
            for t, old in zip((c.k, c.v, c.ks, c.vs), kept):
                t.put(old)
            sync()
            if how == "eager":
                chain()
            else:
                check(lib.vkhip_graph_launch(g, s))
            check(lib.vkhip_stream_sync(s))
            got.append([t.get() for t in (h, r, att, q, k, slot, pos, now, state, c.gpu_table)])
        for a, b in zip(*got):
            assert torch.equal(a, b)
        assert got[0][7].tolist() == [m + many for m in lens]
        c.table = got[0][9]
        T.check_kv_attention(got[0][2].view(n, many, hq, d).double(), c, got[0][3].view(n, many, hq, d).float(), [m + many for m in lens], "f16", 0.125)
    check(lib.vkhip_graph_destroy(g))
    check(lib.vkhip_stream_destroy(s))


@pytest.mark.parametrize("tiles", [None, 256])
def test_shared_calls_side_by_side_and_replayed(gpu, tiles):
    """Two calls under way on streams of their own, and both as graphs, give bit for bit what each gives alone, with
    workspaces that hold anything."""
    lib, page, heads, d, many, t = V.vkhip(), 64, 2, 128, 60, 2
    calls = []
    for seed in (31, 32):
        c, lens, cu = shared_cache([many], [1024], [t + b % 70 for b in range(many)], page, heads, d, seed=seed)
        widen(c, 4 * t, tiles)
        q = rand(seed, many, t, 4 * heads, d).half()
        alone = shared_attention(c, q.float(), lens, cu, [1024], "f16", 0.09)
        desc = V.KvAttentionDesc(q_heads=4 * heads, q_tokens=t, dtype=0, max_len=0, scale=0.09, q_row=4 * heads * d, q_head=d, o_row=4 * heads * d, o_head=d)
        cd, dq, n, dc, dp, out = c.desc(), Dev(q), ints(lens), ints(cu), ints([1024]), full((many, t, 4 * heads, d), 7.0, torch.float16)
        p = V.KvPrefix(cu=dc.data_ptr(), tokens=dp.data_ptr(), groups=1, max_tokens=0, max_tail=0)
        ws, s, g = workspace(lib.vkhip_kv_attention_shared_workspace_bytes(R(desc), R(cd), R(p))), ctypes.c_void_p(), ctypes.c_void_p()
        check(lib.vkhip_stream_create(ctypes.byref(s)))
        calls.append((alone, desc, cd, p, dq, n, out, ws, s, g, (c, dc, dp)))
    sync()

    def launch(call):
        _, desc, cd, p, dq, n, out, ws, s, _, _ = call
        check(lib.vkhip_kv_attention_shared(R(desc), R(cd), R(p), dq.data_ptr(), n.data_ptr(), out.data_ptr(), ws.data_ptr(), s))

    def same():
        for call in calls:
            check(lib.vkhip_stream_sync(call[8]))
        for alone, *_, out, _, _, _, _ in calls:
            assert torch.equal(out.get().double(), alone)
            out.put(torch.full(out.shape, 7.0, dtype=torch.float16))
        sync()
    for _ in range(3):
        for call in calls:
            launch(call)
        same()
    for call in calls:
        check(lib.vkhip_graph_begin(call[8]))
        launch(call)
        check(lib.vkhip_graph_end(call[8], ctypes.byref(call[9])))
    for _ in range(4):
        for call in calls:
            check(lib.vkhip_graph_launch(call[9], call[8]))
        same()
    for call in calls:
        check(lib.vkhip_graph_destroy(call[9]))
        check(lib.vkhip_stream_destroy(call[8]))
