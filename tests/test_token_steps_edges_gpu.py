"""The operators of a token step at their edges: workspaces past 2^31 parts, long prefixes in wide tiles, value scales at
the ends of the number range, launches of very many groups, pages that several sequences name. Against float64, with the
bounds of test_token_steps_gpu.py."""
import copy
import ctypes

import pytest

import test_token_steps_gpu as S
import test_tokens_gpu as T
import vknn_amd as V
from test_tokens_gpu import Dev, full, ints, rand, sync
from vknn_amd import DeviceBuffer, check

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
R = ctypes.byref


class Shared:
    """A call of the attention behind shared prefixes whose workspace says how the host has cut it."""

    def __init__(self, c, q, lens, cu, prefixes, dtype, scale, **hints):
        (self.dt, code, _), (b, t, hq, d) = T.DT[dtype], q.shape
        self.c, self.q, self.lens, self.dtype, self.scale, self.shape = c, q, lens, dtype, scale, (b, t, hq, d)
        self.desc = V.KvAttentionDesc(q_heads=hq, q_tokens=t, dtype=code, scale=scale, q_row=hq * d, q_head=d, o_row=hq * d, o_head=d)
        self.cd, self.keep = c.desc(), [ints(cu), ints(prefixes)]
        self.prefix = V.KvPrefix(cu=self.keep[0].data_ptr(), tokens=self.keep[1].data_ptr(), groups=len(cu) - 1, **hints)
        self.bytes = V.vkhip().vkhip_kv_attention_shared_workspace_bytes(R(self.desc), R(self.cd), R(self.prefix))
        self.rows = hq // c.heads * t
        self.parts = self.bytes // (4 * (d + 2))
        self.splits = self.parts // (b * c.heads * self.rows)  # of a row: of the prefix and of the tail

    def run(self, workspace=None):
        dq, n, out = Dev(self.q.to(self.dt)), ints(self.lens), full(self.shape, 7.0, self.dt)
        ws = workspace or T.workspace(self.bytes)
        sync()
        check(V.vkhip().vkhip_kv_attention_shared(R(self.desc), R(self.cd), R(self.prefix), dq.data_ptr(), n.data_ptr(), out.data_ptr(), getattr(ws, "ptr", None) or ws.data_ptr(), None), "shared")
        sync()
        return out.get().double()

    def check(self, out, ids=None):
        """All sequences, or some of them."""
        ids = list(range(len(self.lens))) if ids is None else ids
        some = copy.copy(self.c)
        some.table = self.c.table[ids]
        T.check_kv_attention(out[ids], some, self.q[ids], [self.lens[i] for i in ids], self.dtype, self.scale)


def widen_table(c, blocks):
    """The same pages in a table of that many blocks a sequence."""
    table = torch.full((c.batch, blocks), -1, dtype=torch.int32)
    table[:, :c.blocks] = c.table
    c.table, c.blocks, c.gpu_table = table, blocks, Dev(table)


def test_shared_more_than_2_31_parts(gpu):
    """A table so wide that a workspace holds more parts than 31 bits number: the last sequence's rows have theirs behind
    the 2^31st. (The workspace, 86 GB, is not cleared: what is read of it has been written.)"""
    many, t, hq, d = 128, 64, 64, 8
    c, lens, cu = S.shared_cache([many], [128], [1 + b % 60 for b in range(many)], 64, 1, d, seed=21)
    widen_table(c, 1 << 20)
    q = rand(22, many, t, hq, d).half().float()
    call = Shared(c, q, lens, cu, [128], "f16", 0.35, max_tail=64)
    assert call.parts > 1 << 31 and (many - 1) * call.rows * call.splits < 1 << 31
    ws = DeviceBuffer(call.bytes)
    out = call.run(ws)
    del ws
    call.check(out, [0, 1, many - 2, many - 1])


@pytest.mark.parametrize("many,tiles,page,d", [(4, None, 64, 64), (60, 128, 64, 64), (60, 256, 64, 128), (60, 128, 32, 64), (20, 128, 32, 128), (60, 256, 32, 128), (20, 128, 64, 128)])
@pytest.mark.parametrize("small,large", [(2.0 ** -60, 2.0 ** 30), (2.0 ** -70, 2.0 ** 70), (2.0 ** -100, 2.0 ** 90), (2.0 ** -100, 1.0), (1.0, 3e37 * 16)])
def test_shared_value_scales_at_both_ends(gpu, many, tiles, page, d, small, large):
    """A prefix whose pages have value scales 2^90 to 2^230 apart, all but the last the small ones: sequences that end in
    front of the last page have what a call without it gives, and those that see it no NaN. Scales are put at most at 4e37
    to 3e38, past 2^126 (values of which bf16 has no numbers: those sequences are compared in front of it alone)."""
    c, lens, cu = S.shared_cache([many], [512], [3] * many, page, 1, d, seed=23)
    for b in range(many):
        c.table[b] = c.table[0]
    c.gpu_table.put(c.table)
    S.widen(c, 4, tiles)
    vs = c.vs.get()
    first, last = c.table[0, :512 // page - 1].long(), int(c.table[0, 512 // page - 1])
    vs[first] *= small
    vs[last] = (vs[last].clamp(max=0.5).double() * large).float()  # the factor alone may be past fp32's largest number
    c.vs.put(vs)
    assert (vs[first] > 2.0 ** -116).all() and torch.isfinite(vs[last]).all()
    end = 512 - page
    lens = [[end, end - 1, 1, 65, 300, 512, 500, 2][b % 8] for b in range(many)]
    q = rand(24, many, 1, 4, d).bfloat16().float()
    call = Shared(c, q, lens, cu, [512], "bf16", 0.125)
    out = call.run()
    seen = [b for b in range(many) if lens[b] > end]
    call.check(out, [b for b in range(many) if b not in seen])
    assert not torch.isnan(out[seen]).any()
    if large < 1e30:
        call.check(out, seen)


def filled(batch, blocks, page, d, seed):
    """A cache of one head whose pages hold any bytes, with scales as of ordinary rows."""
    c = T.Cache(batch, blocks, page, 1, d, seed)
    for i, scales in enumerate((c.ks, c.vs)):
        scales.put(torch.rand(scales.shape, generator=torch.Generator().manual_seed(seed + i)) * 0.02 + 0.005)
    return c


# groups that together have more than 65535 blocks of 32 rows, and ones whose wide tiles would be that many; more groups
# than sequences: those of three have four empty ones behind them
@pytest.mark.parametrize("batch,hq,t,sizes,height", [(32000, 1, 32, [1] * 7 + [3, 0, 0, 0, 0], 32), (16000, 8, 64, [8], 128)])
def test_shared_very_many_groups(gpu, batch, hq, t, sizes, height):
    page, d, cu = 32, 8, [0]
    while cu[-1] < batch:
        cu += [min(batch, cu[-1] + sum(sizes[:i + 1])) for i in range(len(sizes))]
    c = filled(batch, 3, page, d, 25)
    for lo, hi in zip(cu, cu[1:]):
        if hi - lo > 1:
            c.table[lo:hi, 0] = c.table[lo, 0]
    c.gpu_table.put(c.table)
    lens = [page + 1 + b % 63 for b in range(batch)]
    q = rand(26, batch, t, hq, d).half().float()
    call = Shared(c, q, lens, cu, [page * (g % 9 > 0) for g in range(len(cu) - 1)], "f16", 0.35, max_tokens=page, max_tail=70)
    assert batch * hq * t // height + len(cu) - 1 > 65535
    out = call.run(DeviceBuffer(call.bytes))
    call.check(out, [0, 1, 7, 8, 9, 10, batch // 2, batch - 9, batch - 2, batch - 1])


def test_reserve_of_no_sequences(gpu):
    """The sums have one entry, which is 0; the list, where there is one, stays."""
    for pool in (V.KvPool(), None):
        free, state, cu, pos = ints([3, 1, 2, 0]), ints([4, 9]), ints([-9, -9]), ints([-9])
        pool = pool or V.KvPool(free=free.data_ptr(), state=state.data_ptr(), capacity=4)
        cache = V.KvCache(pages=4, page_tokens=64, kv_heads=1, head_dim=64, batch=0, max_blocks=2)
        sync()
        check(V.vkhip().vkhip_kv_reserve(R(cache), R(pool), None, None, 1, cu.data_ptr(), None, pos.data_ptr(), None, None))
        sync()
        assert cu.get().tolist() == [0, -9] and pos.get().tolist() == [-9]
        assert free.get().tolist() == [3, 1, 2, 0] and state.get().tolist() == [4, 9]


@pytest.mark.parametrize("near", [False, True])
def test_rotary_small_angles_keep_their_digits(gpu, near):
    """The pair (1, 0) becomes (cos, sin): a slow pair's sine is good to a few units of itself, not of the turn. The float of
    the angle is rounded from its halves, their factors and their sum (4 * 2^-24 of itself), the series in fp32 (another 3), its
    product and the output (1 each); 9 * 2^-24 in all, beside what a frequency rounded to 2^-64 turns adds a position."""
    at, n, theta = [1, -1, 3, 7, -20, 1000, 4096, -65537, 200000, 2 ** 24 + 1], 64, 1e6
    q = torch.zeros(len(at), 1, 2 * n)
    q[:, :, 0:2 * n:2 if near else 1][:, :, :n] = 1.0
    out, _ = S.rotary(q, None, [at], sections=[n], dtype="f32", near=near, theta=theta)
    sine = out[:, 0, 1::2] if near else out[:, 0, n:]
    cosine = out[:, 0, 0::2] if near else out[:, 0, :n]
    pos = torch.tensor(at, dtype=torch.float64)[:, None]
    angle = pos * theta ** (-torch.arange(n, dtype=torch.float64) / n)
    slow = angle.abs() < 0.75
    assert slow.sum() > 300 and (angle[slow].abs() < 1e-5).any()
    off = (sine.double() - torch.sin(angle)).abs() / (9 * S.F32 * torch.sin(angle).abs() + pos.abs() * 2.0 ** -62 + 1e-38)
    assert off[slow].max() <= 1, off[slow].max()
    assert ((cosine.double() - torch.cos(angle)).abs()[slow] <= 9 * S.F32).all()


@pytest.mark.parametrize("theta", [0.5, 1e-3, 2e-6])
def test_rotary_theta_under_one(gpu, theta):
    """Frequencies that rise from 1: whole turns a position."""
    q = rand(31, 70, 2, 64)
    pos = [list(range(-20, 50)), list(range(3, 700, 10))]
    how = dict(sections=[20, 12], dtype="f32", theta=theta)
    out, _ = S.rotary(q, None, pos, **how)
    S.check_rotary(out, q, pos, **how)


def test_pages_of_a_shared_prefix_go_back_once(gpu):
    """Members of a group end one after the other, the first one first, and draft tokens are taken back between: all but the
    last keep the shared prefix, whose pages then come back with the last one, and the list never names a page twice."""
    page, shared, batch = 32, 3, 5
    p = S.Pool(batch, 8, page, 40, seed=9)
    prefix = shared * page
    now = p.reserve([0] * batch, [prefix] + [0] * (batch - 1), prefix)
    for b in range(1, batch):  # the program names the first one's pages for the others
        p.table[b][:shared] = p.table[0][:shared]
    p.gpu_table.put(torch.tensor(p.table, dtype=torch.int32))
    lens = p.reserve([prefix] * batch, [5, 70, 33, 1, 64], 173)
    left = list(range(batch))
    for b in (0, 3, 1, 4, 2):
        drafts = [3 if i in left else 0 for i in range(batch)]
        now = p.reserve(lens, drafts, sum(drafts))
        p.release(now, lens)
        left.remove(b)
        keep = [n if i != b else prefix if left else 0 for i, n in enumerate(lens)]
        p.release(lens, keep)
        lens = [n if i in left else 0 for i, n in enumerate(keep)]  # what is kept of an ended one's row is the others'
        held = {e for i in left for e in p.table[i] if e >= 0}
        assert len(set(p.free)) == len(p.free) and not held & set(p.free) and len(held) + len(p.free) == 40
    # the rows of the table are free for others, whatever they still name
    now = p.reserve([0] * batch, [2 * page] * batch, 2 * page * batch)
    taken = [e for row in p.table for e in row[:2]]
    assert len(set(taken)) == 2 * batch and not set(taken) & set(p.free)


def test_steps_of_drafts_behind_a_shared_prefix(gpu):
    """Steps of drafted tokens as they would be run: pages, rows into the cache, attention, the rejected tokens' pages back;
    the first two eager, the others replays of one graph, with the program's lengths and rows put in between."""
    lib, page, hkv, hq, d, n, drafts, pre = V.vkhip(), 64, 2, 4, 64, 5, 4, 128
    c, lens, cu = S.shared_cache([n], [pre], [63, 1, 62, 100, 125], page, hkv, d, seed=12, blocks=8)
    count = [-(-m // page) for m in lens]
    used = {int(v) for b in range(n) for v in c.table[b, :count[b]]}
    free = [i for i in range(c.pages) if i not in used][:14]
    for b in range(n):
        c.table[b, count[b]:] = -1
    c.gpu_table.put(c.table)
    rows = n * drafts
    q, att = full((rows, hq * d), 0.0, torch.float16), full((rows, hq * d), 9.0, torch.float16)
    k, v = (full((rows, hkv * d), 0.0, torch.float16) for _ in range(2))
    was, add, now, keep, dcu = ints(lens), ints([drafts] * n), ints([0] * n), ints([0] * n), ints([0] * (n + 1))
    dfree, state, dc, dp = ints(free), ints([len(free), 0]), ints(cu), ints([pre])
    pool, cd = V.KvPool(free=dfree.data_ptr(), state=state.data_ptr(), capacity=len(free)), c.desc()
    kr = V.KvRows(dtype=0, total=rows, k_row=hkv * d, k_head=d, v_row=hkv * d, v_head=d)
    ad = V.KvAttentionDesc(q_heads=hq, q_tokens=drafts, dtype=0, max_len=page * 8, scale=0.125, q_row=hq * d, q_head=d, o_row=hq * d, o_head=d)
    pf = V.KvPrefix(cu=dc.data_ptr(), tokens=dp.data_ptr(), groups=1, max_tokens=pre, max_tail=300)
    ws, s, g = T.workspace(lib.vkhip_kv_attention_shared_workspace_bytes(R(ad), R(cd), R(pf))), ctypes.c_void_p(), ctypes.c_void_p()
    check(lib.vkhip_stream_create(ctypes.byref(s)))

    def chain():
        check(lib.vkhip_kv_reserve(R(cd), R(pool), was.data_ptr(), add.data_ptr(), rows, dcu.data_ptr(), now.data_ptr(), None, None, s))
        check(lib.vkhip_kv_append(R(cd), R(kr), k.data_ptr(), v.data_ptr(), dcu.data_ptr(), was.data_ptr(), s))
        check(lib.vkhip_kv_attention_shared(R(ad), R(cd), R(pf), q.data_ptr(), now.data_ptr(), att.data_ptr(), ws.data_ptr(), s))
        check(lib.vkhip_kv_release(R(cd), R(pool), now.data_ptr(), keep.data_ptr(), s))
    check(lib.vkhip_graph_begin(s))
    chain()
    check(lib.vkhip_graph_end(s, ctypes.byref(g)))
    for i in range(7):
        taken = [(b + i) % (drafts + 1) for b in range(n)]  # none, some or all of the drafts
        kept = [m + t for m, t in zip(lens, taken)]
        was.put(torch.tensor(lens, dtype=torch.int32))
        keep.put(torch.tensor(kept, dtype=torch.int32))
        for t, salt in ((q, 1), (k, 2), (v, 3)):
            t.put(rand(40 + 3 * i + salt, *t.shape).half())
        sync()
        if i < 2:
            chain()
        else:
            check(lib.vkhip_graph_launch(g, s))
        check(lib.vkhip_stream_sync(s))
        table = c.table.clone()
        for b in range(n):  # the pages as the attention had them
            for j in range(-(-lens[b] // page), -(-(lens[b] + drafts) // page)):
                table[b, j] = free.pop()
        c.table = table.clone()
        T.check_kv_attention(att.get().view(n, drafts, hq, d).double(), c, q.get().view(n, drafts, hq, d).float(), [m + drafts for m in lens], "f16", 0.125)
        back = []
        for b in range(n):
            for j in range(-(-kept[b] // page), -(-(lens[b] + drafts) // page)):
                back.append(int(table[b, j]))
                table[b, j] = -1
        free += back[::-1]
        c.table, lens = table, kept
        assert torch.equal(c.gpu_table.get(), table) and state.get().tolist() == [len(free), 0] and dfree.get().tolist()[:len(free)] == free
    check(lib.vkhip_graph_destroy(g))
    check(lib.vkhip_stream_destroy(s))


def long_cache(heads, d, page, tokens, many, tail, seed):
    """One prefix of that many tokens for all, a page or two behind it for each; any bytes, scales as of ordinary rows, so
    that nothing is appended and the table alone is large."""
    blocks = tokens // page + 2
    c = T.Cache.__new__(T.Cache)
    c.page, c.heads, c.d, c.dp, c.batch, c.blocks, c.pages = page, heads, d, V.vkhip().vkhip_kv_row(d), many, blocks, tokens // page + 2 * many
    g = torch.Generator().manual_seed(seed)
    names = torch.randperm(c.pages, generator=g).int()
    c.table = torch.empty((many, blocks), dtype=torch.int32)
    c.table[:, :-2] = names[:blocks - 2]
    c.table[:, -2:] = names[blocks - 2:].view(many, 2)
    c.gpu_table = Dev(c.table)
    c.k, c.v = (Dev(torch.randint(-127, 128, (c.pages, heads) + shape, generator=g, dtype=torch.int8)) for shape in ((page, c.dp), (c.dp, page)))
    c.ks, c.vs = (Dev(torch.rand((c.pages, heads), generator=g) * 0.02 + 0.005) for _ in range(2))
    return c, [tokens + tail(b) for b in range(many)]


# Tiles of 128 rows for 64 channels (512 places on the card) and of 256 for 128 (256): one workgroup takes 256 tiles of 64
# tokens at most, 128 with pages of 32, and as many rows as fill the places leave it all that it may hold.
LONG = [(128, 64, 16384, 1, "f16"), (128, 64, 16384 + 64, 2, "f16"), (128, 64, 32768 - 192, 2, "bf16"), (128, 32, 8192, 1, "f16"), (128, 32, 8192 + 32, 2, "bf16"), (128, 32, 16384 - 32, 2, "f16"),
        (64, 64, 16384, 1, "bf16"), (64, 128, 32768 - 128, 2, "f16"), (64, 32, 8192, 1, "f16"), (64, 32, 16384 + 32, 3, "f16"), (96, 256, 16384, 1, "f16"), (40, 64, 16384 + 128, 2, "f16")]


@pytest.mark.parametrize("d,page,tokens,splits,dtype", LONG)
def test_shared_long_spans_in_wide_tiles(gpu, d, page, tokens, splits, dtype):
    """Workgroups that hold as many tiles as they can: full lists of pages, accumulation over hundreds of tiles, and spans that
    the limit splits although the rows alone fill the card. Some sequences end inside the prefix, at the last tile's first
    and last token among them."""
    heads, many, hq, t = 4, 32, 64, 32  # 512 rows a sequence, 16384 of a group and head
    c, lens = long_cache(heads, d, page, tokens, many, lambda b: 30 + b, d + page)
    span = -(-(tokens // 64) // splits) * 64
    lens[3:9] = [t, tokens, tokens - 1, tokens - 63, min(tokens, span + 5), min(tokens, span) - 1]
    q = rand(41, many, t, hq, d).to(T.DT[dtype][0]).float()
    call = Shared(c, q, lens, [0, many], [tokens], dtype, d ** -0.5, max_tokens=tokens, max_tail=80)
    assert call.splits == splits + 1  # the tail has one
    out = call.run(DeviceBuffer(call.bytes))
    # a few heads and rows of some sequences, the keys' sum being long: the bound's terms for weights under fp16's smallest go
    # by the number of tokens, as everywhere
    for b in (0, 3, 4, 5, 6, 7, 8, many - 1):
        (kq, ks), (vq, vs) = c.bytes_of(b, lens[b])
        for h in (0, hq - 1):
            one = h * heads // hq
            k, v = ((x[:, one:one + 1].double() * s[:, one:one + 1, None]) for x, s in ((kq, ks), (vq, vs)))
            extra = 0.0 if dtype == "f16" else d * 2.0 ** -25
            T.check_attention(out[b][:, h:h + 1], q[b][:, h:h + 1].double(), k, v, [t], [lens[b]], True, dtype, d ** -0.5, weights_dtype="f16", extra=extra)


@pytest.mark.parametrize("d,hq", [(128, 64), (64, 512)])
def test_shared_wide_tiles_of_a_cut_prefix(gpu, d, hq):
    """max_tokens under the prefix, on a page's border and not: wide tiles take it up to there, each sequence the rest."""
    heads, many, tokens = 8, 64, 4096
    c, lens = long_cache(heads, d, 64, tokens, many, lambda b: 1 + b, 42)
    q = rand(43, many, 1, hq, d).half().float()
    for most in (tokens - 64, tokens - 1, tokens // 2 + 640 + 31):
        assert heads * many * hq // heads * (most // 64 * 64) > (1 << 23 if d == 128 else 3 << 24)
        call = Shared(c, q, lens, [0, many], [tokens], "f16", d ** -0.5, max_tokens=most, max_tail=tokens - most + 64 + many)
        call.check(call.run(), [0, 17, many - 1])


def test_shared_wide_tiles_of_many_groups(gpu):
    """More groups than a wave has lanes, each with rows for wide tiles, empty ones between them."""
    heads, d, hq, t, page = 4, 128, 32, 4, 64
    sizes = [0 if g % 11 == 5 else 1 + g % 6 for g in range(90)]
    prefixes = [page * (1 + g % 9) for g in range(90)]
    c, lens, cu = S.shared_cache(sizes, prefixes, [t + b % 60 for b in range(sum(sizes))], page, heads, d, seed=44)
    assert heads * sum(sizes) * hq // heads * t * max(prefixes) > 1 << 24 and sum(sizes) * hq // heads * t // 90 > 64
    q = rand(45, len(lens), t, hq, d).half().float()
    call = Shared(c, q, lens, cu, prefixes, "f16", d ** -0.5, max_tokens=max(prefixes), max_tail=64)
    call.check(call.run(), list(range(0, len(lens), 7)) + [len(lens) - 1])
