"""What a step of a token model over many requests needs beside its products and its cache, as cases that can be
timed and checked: rotary positions with several axes, pages and positions of the step's rows from lengths on the
GPU, attention over the 8-bit cache where sequences share a prefix, and the norms before and after a block with its
gate and residual. Each case is one call of the kernel library's C ABI (include/vkhip.h), or the pair of calls that
belong together, on tensors that sit on the GPU and on the program's current stream; the plain forms are the same
operators in elementary tensor operations, in 32 bits (angles in 64).
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
DT_CODE = {"f16": 0, "bf16": 1, "f32": 2}
NORM = {"none": 0, "rms": 1, "layer": 2}
EPS = 1e-5


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # A decode step's rows: one token of 64 requests, grouped heads, positions far behind images and text.
        dict(name="rope_step", op="rope", rows=64, frames=0, side=0, hq=32, hk=8, d=128, rot=128, sections="16,24,24", deal=False, spectra=False, near=False, theta=1e6, dtype="bf16"),
        # Eight images' 75 x 75 maps as tokens: two axes with a spectrum each, neighbouring channels in pairs.
        dict(name="rope_images", op="rope", rows=45000, frames=1, side=75, hq=16, hk=16, d=64, rot=64, sections="16,16", deal=False, spectra=True, near=True, theta=1e4, dtype="f16"),
        # Frames of a video as one long prompt, axes dealt to the pairs in turn: half a gigabyte in and out.
        dict(name="rope_video", op="rope", rows=50176, frames=16, side=56, hq=32, hk=8, d=128, rot=128, sections="24,20,20", deal=True, spectra=False, near=False, theta=1e6, dtype="bf16"),
        # The ordinary step of 256 requests: a token each, a new page for the few that start one, and these back.
        dict(name="pages_step", op="pages", b=256, lo=1, hi=4000, new_lo=1, new_hi=1, page=64),
        # Prompts of 64 requests behind what they hold: a quarter of a million rows.
        dict(name="pages_prompt", op="pages", b=64, lo=0, hi=2000, new_lo=100, new_hi=8000, page=64),
        # Four questions about one image: latency.
        dict(name="shared_b4", op="shared", groups=1, n_lo=4, n_hi=4, pre_lo=1024, pre_hi=1024, lo=1, hi=100, t=1, hq=32, hkv=8, d=128, page=64, dtype="f16"),
        # The ordinary step: 64 requests behind one prompt, with answers of different lengths.
        dict(name="shared_b64", op="shared", groups=1, n_lo=64, n_hi=64, pre_lo=4096, pre_hi=4096, lo=1, hi=600, t=1, hq=32, hkv=8, d=128, page=64, dtype="f16"),
        # Groups of different sizes and prefixes, drafted tokens, smaller heads and pages.
        dict(name="shared_groups", op="shared", groups=7, n_lo=1, n_hi=40, pre_lo=0, pre_hi=9000, lo=3, hi=800, t=3, hq=16, hkv=4, d=64, page=32, dtype="bf16"),
        # Many requests behind a long document: where the matrix units count.
        dict(name="shared_long", op="shared", groups=1, n_lo=256, n_hi=256, pre_lo=32768, pre_hi=32768, lo=200, hi=2000, t=1, hq=32, hkv=8, d=128, page=64, dtype="bf16"),
        # Between two blocks of a decode step.
        dict(name="norm_step", op="norm", rows=64, each=64, dim=4096, post="rms", pre="rms", gate=False, mod=False, bias=False, dtype="bf16"),
        # Eight images' 40 x 40 tokens of an odd width: a gate, scale and shift for each image around a layer norm.
        dict(name="norm_images", op="norm", rows=12800, each=1600, dim=1100, post="none", pre="layer", gate=True, mod=True, bias=False, dtype="f16"),
        # A video's tokens: a norm on both sides and a gate for each frame, 800 MB in and out.
        dict(name="norm_video", op="norm", rows=50176, each=3136, dim=2048, post="rms", pre="rms", gate=True, mod=False, bias=False, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {op: max(work(c)["flops" if op == "shared" else "bytes"] for c in listed() if c["op"] == op) for op in ("rope", "pages", "shared", "norm")}
    op = rng.choice(["rope", "rope", "pages", "shared", "shared", "shared", "shared", "norm", "norm"])
    while True:
        if op == "rope":
            # 1 to 60000 rows of text, images or video; heads of 16 to 256, all of their channels turned or some
            axes = rng.choice([1, 2, 3])
            unit = rng.choice([1, 2, 4, 8])
            parts = [unit * rng.randint(1, max(1, 64 // unit // axes)) for _ in range(axes)]
            rot = 2 * sum(parts)
            d = rng.choice([x for x in (16, 32, 40, 64, 72, 80, 96, 128, 160, 192, 256) if x >= rot])
            side = _log(rng, 2, 80)
            frames = rng.choice([0, 1, 1, _log(rng, 2, 32)])
            rows = _log(rng, 1, 4000) if frames == 0 else frames * side * side * _log(rng, 1, 8)
            hk = rng.choice([0, 1, 2, 4, 8, 16])
            case = dict(op=op, rows=rows, frames=frames, side=side if frames else 0, hq=max(1, hk) * rng.choice([1, 2, 4]), hk=hk, d=d, rot=rot, sections=",".join(map(str, parts)),
                        deal=rng.random() < 0.4, spectra=rng.random() < 0.4, near=rng.random() < 0.4, theta=rng.choice([1e4, 5e5, 1e6]), dtype=rng.choice(["f16", "bf16", "bf16", "f32"]))
        elif op == "pages":
            new = rng.choice([1, _log(rng, 2, 8), _log(rng, 2, 8000)])
            case = dict(op=op, b=_log(rng, 1, 2048), lo=0, hi=_log(rng, 1, 9000), new_lo=rng.randint(0, new), new_hi=new, page=rng.choice([32, 64, 128, 256]))
        elif op == "shared":
            # 1 to 256 sequences in 1 to 12 groups, prefixes up to 32768 tokens, up to 2000 of a sequence's own
            hkv, hi, pre = rng.choice([1, 2, 4, 8]), _log(rng, 8, 2000), _log(rng, 64, 32768)
            groups, n = _log(rng, 1, 12), _log(rng, 1, 256)
            case = dict(op=op, groups=groups, n_lo=max(1, int(n * rng.random())), n_hi=n, pre_lo=int(pre * rng.choice([0, rng.random(), 1])), pre_hi=pre, lo=rng.randint(1, hi), hi=hi,
                        t=rng.choice([1, 1, 1, 2, 3, 5]), hq=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv, d=rng.choice([64, 80, 96, 128, 128]), page=rng.choice([32, 64, 64, 128]), dtype=rng.choice(["f16", "bf16"]))
        else:
            # 1 to 50000 rows of 16 to 16384 values, odd widths among them
            dim = _log(rng, 16, 16384)
            dim = rng.choice([dim, dim // 8 * 8, dim // 128 * 128 or 64])
            each = _log(rng, 1, 4000)
            case = dict(op=op, rows=_log(rng, 1, 50000), each=each, dim=dim, post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["rms", "layer"]), gate=rng.random() < 0.6,
                        mod=rng.random() < 0.5, bias=rng.random() < 0.3, dtype=rng.choice(["f16", "bf16", "bf16", "f32"]))
        w = work(case)
        if w["flops" if op == "shared" else "bytes"] <= most[op] and w["bytes"] <= 1.3e9 and (op != "shared" or sum(_sizes(case)) <= 512):
            return case


# ------------------------------------------------------------------------------------ sizes and inputs
def _lengths(lo, hi, b, salt):
    """b lengths from lo to hi, both ends among them, in a mixed order; fixed by the case alone."""
    r = np.random.default_rng([lo, hi, b, salt])
    a = r.integers(lo, hi + 1, size=b)
    a[0] = hi
    if b > 1:
        a[1] = lo
    return [int(v) for v in r.permutation(a)]


def _sections(c):
    return [int(v) for v in c["sections"].split(",")]


def _axis_of(c):
    """The axis of each pair of channels and its number among the axis's pairs."""
    left, got = _sections(c), []
    if c["deal"]:
        had = [0] * len(left)
        while any(left):
            for a in range(len(left)):
                if left[a]:
                    got.append((a, had[a]))
                    left[a], had[a] = left[a] - 1, had[a] + 1
    else:
        got = [(a, i) for a, n in enumerate(left) for i in range(n)]
    return got


def _sizes(c):
    """Sequences of each group."""
    return _lengths(c["n_lo"], c["n_hi"], c["groups"], 5)


def _prefixes(c):
    """Tokens that each group shares, whole pages."""
    return [n // c["page"] * c["page"] for n in _lengths(c["pre_lo"], c["pre_hi"], c["groups"], 6)]


def _tails(c):
    """Tokens of each sequence behind its group's prefix; the step's own are among them."""
    return [max(n, c["t"]) for n in _lengths(c["lo"], c["hi"], sum(_sizes(c)), 7)]


def _dp(d):
    return 64 if d <= 64 else 128


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 131 + salt) & 0x7FFFFFFF)
    return g


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _positions(c, seed):
    """[axes, rows]: (frame, line, column) of a video's rows behind a short text, one number on every axis for text."""
    axes, rows, r = len(_sections(c)), c["rows"], np.random.default_rng([seed & 0x7FFFFFFF, 9])
    if c["frames"] == 0:
        return np.tile(r.integers(0, 200000, size=rows).astype(np.int32), (axes, 1))
    i, side = np.arange(rows), c["side"]
    all3 = np.stack([i // (side * side) % c["frames"], i // side % side, i % side]) + int(r.integers(0, 1000))
    return all3[3 - axes:].astype(np.int32)


def _page_plan(c, seed):
    """Requests that hold lens tokens and get new ones, every page of both given out from a mixed list."""
    page, b = c["page"], c["b"]
    r = np.random.default_rng([seed & 0x7FFFFFFF, 11])
    lens, new = r.permutation(_lengths(c["lo"], c["hi"], b, 1)), r.permutation(_lengths(c["new_lo"], c["new_hi"], b, 2))
    had, blocks = -(-lens // page), -(-(lens + new) // page)
    most = int(had.sum() + (-(-new // page)).sum())  # whichever of them come together
    width, pages = max(1, -(-(c["hi"] + c["new_hi"]) // page)), most + most // 8 + 5
    order = r.permutation(pages).astype(np.int32)
    table = np.full((b, width), -1, np.int32)
    at = pages
    for first, last in ((0 * had, had), (had, blocks)):  # what they hold, then the step's
        for i in range(b):
            n = int(last[i] - first[i])
            table[i, first[i]:last[i]] = order[at - n:at][::-1]
            at -= n
    return dict(lens=lens, new=new, width=width, pages=pages, order=order, left=at, table=table)


def _shared_cache(c, seed):
    """Pages of the groups' prefixes and of the sequences' tails, int8 with scales; tables whose first blocks are shared."""
    page, hkv, d, dp = c["page"], c["hkv"], c["d"], _dp(c["d"])
    sizes, pre, tails = _sizes(c), _prefixes(c), _tails(c)
    of = [g for g, n in enumerate(sizes) for _ in range(n)]
    lens = [pre[g] + n for g, n in zip(of, tails)]
    width = max(-(-n // page) for n in lens)
    total = sum(p // page for p in pre) + sum(-(-n // page) for n in tails) + 1
    order = np.random.default_rng([seed & 0x7FFFFFFF, 5]).permutation(total).astype(np.int32)
    table, at, heads = np.full((len(of), width), -1, np.int32), 0, []
    for p in pre:
        heads.append(order[at:at + p // page])
        at += p // page
    for i, n in enumerate(tails):
        k, m = len(heads[of[i]]), -(-n // page)
        table[i, :k], table[i, k:k + m] = heads[of[i]], order[at:at + m]
        at += m
    g = _gen(seed, 3)
    k = torch.zeros((total, hkv, page, dp), dtype=torch.int8, device="cuda")
    v = torch.zeros((total, hkv, dp, page), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 26) // (hkv * page * d))
    for i in range(0, total, step):  # the values of normally distributed rows whose largest of a page is about four deviations
        e = min(total, i + step)
        k[i:e, :, :, :d] = (torch.randn((e - i, hkv, page, d), generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)
        v[i:e, :, :d, :] = (torch.randn((e - i, hkv, d, page), generator=g, device="cuda") * 32).round_().clamp_(-127, 127).to(torch.int8)
    ks = torch.rand((total, hkv), generator=g, device="cuda") * 0.02 + 0.02
    vs = torch.rand((total, hkv), generator=g, device="cuda") * 0.02 + 0.02
    q = torch.randn((len(of), c["t"], c["hq"], d), generator=_gen(seed, 6), device="cuda").to(DTYPES[c["dtype"]])
    cu = [0] + [int(x) for x in np.cumsum(sizes)]
    return dict(k=k, v=v, ks=ks, vs=vs, q=q, table=torch.from_numpy(table).cuda(), pages=total, width=width, lens=lens, pre=pre, cu=cu, tails=tails)


def _inputs(c, seed):
    """Everything random of a case."""
    op = c["op"]
    if op == "pages":
        return _page_plan(c, seed)
    if op == "shared":
        return _shared_cache(c, seed)
    dt, g = DTYPES[c["dtype"]], _gen(seed, 1)
    if op == "rope":
        # one product of a projection makes query, key and value rows side by side
        hq, hk, d = c["hq"], c["hk"], c["d"]
        qkv = torch.randn((c["rows"], (hq + 2 * hk) * d), generator=g, device="cuda", dtype=dt if dt != torch.float16 else torch.float32).to(dt)
        return dict(q=qkv[:, :hq * d].unflatten(1, (hq, d)), k=qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d)) if hk else None, pos=torch.from_numpy(_positions(c, seed)).cuda())
    rows, dim = c["rows"], c["dim"]
    mods = -(-rows // c["each"])
    # a block's output beside a residual that has grown over many blocks, a few channels of it large
    x = torch.randn((rows, dim), generator=g, device="cuda").to(dt)
    r = torch.randn((rows, dim), generator=g, device="cuda")
    r = (r * (1 + 30 * (torch.rand(dim, generator=g, device="cuda") > 0.99)) + 0.2).to(dt)
    vec = torch.randn((mods, 3 * dim), generator=g, device="cuda").mul_(0.5).to(dt)  # gate, scale and shift of one projection

    def weight():
        return torch.rand(dim, generator=g, device="cuda") + 0.5
    return dict(x=x, r=r, post_w=weight() if c["post"] != "none" else None, pre_w=weight(), bias=torch.randn(dim, generator=g, device="cuda") * 0.2 if c["bias"] else None,
                gate=vec[:, :dim] if c["gate"] else None, scale=vec[:, dim:2 * dim] if c["mod"] else None, shift=vec[:, 2 * dim:] if c["mod"] else None)


# ------------------------------------------------------------------------------------ state and passes
def prepare(case, seed):
    c, d = dict(case), _inputs(case, seed)
    st, op = {"case": c, **d}, c["op"]
    if op == "rope":
        dt, n = DTYPES[c["dtype"]], c["rows"]
        st["out_q"] = torch.empty((n, c["hq"], c["d"]), dtype=dt, device="cuda")
        st["out_k"] = torch.empty((n, c["hk"], c["d"]), dtype=dt, device="cuda") if c["hk"] else None
    elif op == "pages":
        total = int(d["new"].sum())
        st.update(total=total, gpu_lens=_ints(d["lens"]), add=_ints(d["new"]), now=_ints(d["lens"] + d["new"]), gpu_table=torch.from_numpy(d["table"]).cuda(),
                  free=torch.from_numpy(d["order"]).cuda(), state=_ints([d["left"], 0]), cu=torch.zeros(c["b"] + 1, dtype=torch.int32, device="cuda"),
                  pos=torch.zeros(total, dtype=torch.int32, device="cuda"), slot=torch.zeros(total, dtype=torch.int64, device="cuda"))
    elif op == "shared":
        st.update(gpu_lens=_ints(d["lens"]), gpu_cu=_ints(d["cu"]), gpu_pre=_ints(d["pre"]), out=torch.empty_like(d["q"]))
    else:
        st.update(h=torch.empty_like(d["x"]), y=torch.empty_like(d["x"]))
    if own:
        _prepare_own(st)
    torch.cuda.synchronize()
    return st


def _prepare_own(st):
    """The descriptors and the workspace that a program keeps beside its tensors."""
    import vknn_amd as V
    lib, c, op = V.require_gpu(), st["case"], st["case"]["op"]
    st.update(lib=lib, check=V.check)
    ws = 0
    if op == "rope":
        q, k, s = st["q"], st["k"] if c["hk"] else st["q"], (_sections(c) + [0, 0, 0, 0])[:4]
        st["desc"] = V.RotaryDesc(rows=c["rows"], q_heads=c["hq"], k_heads=c["hk"], head_dim=c["d"], rotary_dim=c["rot"], dtype=DT_CODE[c["dtype"]], neighbours=int(c["near"]),
                                  axes=len(_sections(c)), sections=tuple(s), interleaved=int(c["deal"]), spectra=int(c["spectra"]), theta=c["theta"], pos_axis=c["rows"],
                                  q_row=q.stride(0), q_head=q.stride(1), k_row=k.stride(0), k_head=k.stride(1), qo_row=c["hq"] * c["d"], qo_head=c["d"],
                                  ko_row=c["hk"] * c["d"], ko_head=c["d"])
    elif op == "pages":
        st["cache"] = V.KvCache(table=st["gpu_table"].data_ptr(), pages=st["pages"], page_tokens=c["page"], kv_heads=1, head_dim=64, batch=c["b"], max_blocks=st["width"])
        st["pool"] = V.KvPool(free=st["free"].data_ptr(), state=st["state"].data_ptr(), capacity=st["pages"])
    elif op == "shared":
        q = st["q"]
        st["cache"] = V.KvCache(k=st["k"].data_ptr(), v=st["v"].data_ptr(), k_scale=st["ks"].data_ptr(), v_scale=st["vs"].data_ptr(), table=st["table"].data_ptr(),
                                pages=st["pages"], page_tokens=c["page"], kv_heads=c["hkv"], head_dim=c["d"], batch=len(st["lens"]), max_blocks=st["width"])
        st["desc"] = V.KvAttentionDesc(q_heads=c["hq"], q_tokens=c["t"], dtype=DT_CODE[c["dtype"]], max_len=max(st["lens"]), scale=c["d"] ** -0.5,
                                       q_row=q.stride(1), q_head=q.stride(2), o_row=q.stride(1), o_head=q.stride(2))
        st["prefix"] = V.KvPrefix(cu=st["gpu_cu"].data_ptr(), tokens=st["gpu_pre"].data_ptr(), groups=len(st["pre"]), max_tokens=max(st["pre"]), max_tail=max(st["tails"]))
        ws = lib.vkhip_kv_attention_shared_workspace_bytes(ctypes.byref(st["desc"]), ctypes.byref(st["cache"]), ctypes.byref(st["prefix"]))
    else:
        dim = c["dim"]
        st["desc"] = V.ResidualNormDesc(rows=c["rows"], dim=dim, dtype=DT_CODE[c["dtype"]], post=NORM[c["post"]], pre=NORM[c["pre"]], mods=-(-c["rows"] // c["each"]), mod_rows=c["each"],
                                        alpha=0.7, post_eps=EPS, pre_eps=EPS, x_row=dim, r_row=dim, h_row=dim, y_row=dim, mod_row=3 * dim)
    st["ws"] = torch.empty(max(ws, 16), dtype=torch.uint8, device="cuda")


def run(state):
    return (_run_own if own else _run_plain)(state)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _run_own(st):
    lib, op, ref = st["lib"], st["case"]["op"], ctypes.byref
    # the library's NULL is its own stream; 1 is the runtime's handle of the default stream
    s = torch.cuda.current_stream().cuda_stream or 1
    if op == "rope":
        st["check"](lib.vkhip_rotary(ref(st["desc"]), st["pos"].data_ptr(), None, st["q"].data_ptr(), _ptr(st["k"]), st["out_q"].data_ptr(), _ptr(st["out_k"]), s), "rotary")
        return [st["out_q"], st["out_k"]] if st["case"]["hk"] else [st["out_q"]]
    if op == "pages":
        st["check"](lib.vkhip_kv_release(ref(st["cache"]), ref(st["pool"]), st["now"].data_ptr(), st["gpu_lens"].data_ptr(), s), "kv_release")
        st["check"](lib.vkhip_kv_reserve(ref(st["cache"]), ref(st["pool"]), st["gpu_lens"].data_ptr(), st["add"].data_ptr(), st["total"], st["cu"].data_ptr(), st["now"].data_ptr(),
                                         st["pos"].data_ptr(), st["slot"].data_ptr(), s), "kv_reserve")
        return [st["gpu_table"], st["free"], st["state"], st["cu"], st["now"], st["pos"], st["slot"]]
    if op == "shared":
        st["check"](lib.vkhip_kv_attention_shared(ref(st["desc"]), ref(st["cache"]), ref(st["prefix"]), st["q"].data_ptr(), st["gpu_lens"].data_ptr(), st["out"].data_ptr(),
                                                  st["ws"].data_ptr(), s), "kv_attention_shared")
        return [st["out"]]
    st["check"](lib.vkhip_residual_norm(ref(st["desc"]), st["x"].data_ptr(), st["r"].data_ptr(), _ptr(st["post_w"]), None, _ptr(st["gate"]), st["pre_w"].data_ptr(), _ptr(st["bias"]),
                                        _ptr(st["scale"]), _ptr(st["shift"]), None, st["h"].data_ptr(), st["y"].data_ptr(), s), "residual_norm")
    return [st["h"], st["y"]]


def _run_plain(st):
    return {"rope": _plain_rope, "pages": _plain_pages, "shared": _plain_shared, "norm": _plain_norm}[st["case"]["op"]](st)


def _plain_rope(st):
    c = st["case"]
    parts, of = _sections(c), _axis_of(c)
    freq = [c["theta"] ** -(j / parts[a] if c["spectra"] else i / len(of)) for i, (a, j) in enumerate(of)]
    angle = st["pos"][[a for a, _ in of]].t().double() * torch.tensor(freq, dtype=torch.float64, device="cuda")
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def turn(x):
        y, n = x.float(), len(of)
        a, b = (y[..., 0:2 * n:2], y[..., 1:2 * n:2]) if c["near"] else (y[..., :n], y[..., n:2 * n])
        p, q = a * cos - b * sin, b * cos + a * sin
        return torch.cat([torch.stack([p, q], -1).flatten(-2) if c["near"] else torch.cat([p, q], -1), y[..., 2 * n:]], -1).to(x.dtype)
    return [turn(st["q"]), turn(st["k"])] if c["hk"] else [turn(st["q"])]


def _plain_pages(st):
    page, table, free, state = st["case"]["page"], st["gpu_table"], st["free"], st["state"]
    lens, add, n = st["gpu_lens"].long(), st["add"].long(), free.numel()
    block = torch.arange(table.shape[1], device="cuda")
    # the pages behind what is kept, in order, go onto the list, the first of them last
    back = (block >= (lens + page - 1)[:, None] // page) & (block < (st["now"].long() + page - 1)[:, None] // page) & (table >= 0)
    rank = back.flatten().cumsum(0) - 1
    count = state[0] + rank[-1] + 1
    held = torch.cat([free, free[:1]])
    held[torch.where(back.flatten(), count - 1 - rank, n)] = table.flatten()
    free.copy_(held[:n])
    table.masked_fill_(back, -1)
    # and the blocks that the new tokens need take pages from its end
    want = (block >= (lens + page - 1)[:, None] // page) & (block < (lens + add + page - 1)[:, None] // page)
    rank = (want.flatten().cumsum(0) - 1).view(want.shape)
    total, at = rank[-1, -1] + 1, count - 1 - rank
    table.copy_(torch.where(want, torch.where(at >= 0, free[at.clamp(0, n - 1)], -1), table))
    state.copy_(torch.stack([(count - total).clamp(min=0), state[1] + (total - count).clamp(min=0)]))
    now = lens + add
    cu = torch.cat([torch.zeros_like(add[:1]), add.cumsum(0)])
    row = torch.arange(st["total"], device="cuda")
    seq = torch.searchsorted(cu[1:], row, right=True)
    pos = lens[seq] + row - cu[seq]
    name = table[seq, pos // page].long()
    return [table, free, state, cu.int(), now.int(), pos.int(), torch.where(name >= 0, name * page + pos % page, -1)]


def _plain_shared(st):
    c = st["case"]
    page, hkv, d, t, hq = c["page"], c["hkv"], c["d"], c["t"], c["hq"]
    out, rows = torch.empty_like(st["q"]), c["hq"] // c["hkv"] * c["t"]

    def values(ids):  # blocks' keys and values: [..., hkv, tokens, d]
        k = st["k"][ids][..., :d].float() * st["ks"][ids][..., None, None]
        v = st["v"][ids][..., :d, :].float().transpose(-1, -2) * st["vs"][ids][..., None, None]
        return [x.transpose(-4, -3).flatten(-3, -2) for x in (k, v)]
    for at, end, pre in zip(st["cu"], st["cu"][1:], st["pre"]):
        n, lens = end - at, st["gpu_lens"][at:end]
        # rows of a key/value head: sequence, query head of the group, token
        q = st["q"][at:end].float().view(n, t, hkv, hq // hkv, d).permute(2, 0, 3, 1, 4).reshape(hkv, n, rows, d) * d ** -0.5
        blocks = -(-max(st["lens"][at:end]) // page)
        k, v = values(st["table"][at:end, pre // page:blocks].long().clamp(min=0))
        see = (lens[:, None] - t + torch.arange(t, device="cuda")).repeat(1, hq // hkv)  # the last position that a row sees
        s = torch.matmul(q.transpose(0, 1), k.transpose(-1, -2))  # [n, hkv, rows, tokens]
        s.masked_fill_(torch.arange(pre, blocks * page, device="cuda") > see[:, None, :, None], -math.inf)
        top = s.amax(-1)
        if pre:
            pk, pv = values(st["table"][at, :pre // page].long())
            ps = torch.matmul(q.reshape(hkv, n * rows, d), pk.transpose(-1, -2))
            top = torch.maximum(top, ps.amax(-1).view(hkv, n, rows).transpose(0, 1))
            ps.sub_(top.transpose(0, 1).reshape(hkv, n * rows, 1)).exp_()
        s.sub_(top[..., None]).exp_()
        total, o = s.sum(-1), torch.matmul(s, v)
        if pre:
            total = total + ps.sum(-1).view(hkv, n, rows).transpose(0, 1)
            o += torch.matmul(ps, pv).view(hkv, n, rows, d).transpose(0, 1)
        out[at:end] = (o / total[..., None]).view(n, hkv, hq // hkv, t, d).permute(0, 3, 1, 2, 4).reshape(n, t, hq, d).to(out.dtype)
    return [out]


def _plain_norm(st):
    c = st["case"]

    def norm(z, kind, w, b):
        if kind == "none":
            return z
        if kind == "layer":
            z = z - z.mean(-1, keepdim=True)
        z = z * torch.rsqrt((z * z).mean(-1, keepdim=True) + EPS) * w
        return z if b is None else z + b

    def of_row(v):
        return v.float().repeat_interleave(c["each"], 0)[:c["rows"]]
    f = norm(st["x"].float(), c["post"], st["post_w"], None) * 0.7
    h = st["r"].float() + (f * of_row(st["gate"]) if c["gate"] else f)
    y = norm(h, c["pre"], st["pre_w"], st["bias"])
    if c["mod"]:
        y = y * (1 + of_row(st["scale"])) + of_row(st["shift"])
    return [h.to(st["x"].dtype), y.to(st["x"].dtype)]


# ------------------------------------------------------------------------------------ float64 values
def exact(case, seed):
    c, op = case, case["op"]
    if op == "pages":
        return None
    d = _inputs(case, seed)
    if op == "rope":
        # a pair of channels as a complex number, turned
        turns, n = torch.empty((c["rows"], c["rot"] // 2), dtype=torch.float64, device="cuda"), c["rot"] // 2
        for i, (a, j) in enumerate(_axis_of(c)):
            turns[:, i] = d["pos"][a].double() / math.exp(math.log(c["theta"]) * (j / _sections(c)[a] if c["spectra"] else i / n))
        z, outs = torch.polar(torch.ones_like(turns), turns), []
        for x in [d["q"]] + ([d["k"]] if c["hk"] else []):
            y = x.double()
            for h in range(x.shape[1]):
                one, two = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["near"] else (slice(0, n), slice(n, 2 * n))
                w = torch.complex(y[:, h, one], y[:, h, two]) * z
                y[:, h, one], y[:, h, two] = w.real, w.imag
            outs.append(y)
        return outs
    if op == "norm":
        outs = [torch.empty((c["rows"], c["dim"]), dtype=torch.float64, device="cuda") for _ in range(2)]

        def norm(z, kind, w, b):
            if kind == "rms":
                z = z / (z.square().mean(1, keepdim=True) + EPS).sqrt()
            elif kind == "layer":
                var, mean = torch.var_mean(z, dim=1, keepdim=True, correction=0)
                z = (z - mean) / (var + EPS).sqrt()
            else:
                return z
            return z * w.double() + (0 if b is None else b.double())
        for i in range(0, c["rows"], 8192):  # some rows at a time
            at = torch.arange(i, min(c["rows"], i + 8192), device="cuda")
            m = at // c["each"]
            block = norm(d["x"][at].double(), c["post"], d["post_w"], None)
            h = d["r"][at].double() + 0.7 * (block * d["gate"][m].double() if c["gate"] else block)
            y = norm(h, c["pre"], d["pre_w"], d["bias"])
            outs[0][at] = h
            outs[1][at] = y + y * d["scale"][m].double() + d["shift"][m].double() if c["mod"] else y
        return outs
    page, dim, hkv, t = c["page"], c["d"], c["hkv"], c["t"]
    group, table = c["hq"] // hkv, d["table"].cpu().numpy()
    out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    for b, n in enumerate(d["lens"]):  # a sequence and head at a time, over its whole table
        ids = torch.from_numpy(table[b, :-(-n // page)].astype(np.int64)).cuda()
        see = torch.arange(n, device="cuda")[None] <= torch.arange(n - t, n, device="cuda")[:, None]
        for h in range(hkv):
            k = (d["k"][ids, h].double() * d["ks"][ids, h].double()[:, None, None]).flatten(0, 1)[:n, :dim]
            v = (d["v"][ids, h].double() * d["vs"][ids, h].double()[:, None, None]).transpose(1, 2).flatten(0, 1)[:n, :dim]
            z = torch.einsum("tgc,nc->gtn", d["q"][b, :, h * group:(h + 1) * group].double(), k) / math.sqrt(dim)
            z = torch.where(see, z, -math.inf)
            out[b, :, h * group:(h + 1) * group] = torch.einsum("gtn,nc->tgc", torch.exp(z - torch.logsumexp(z, 2, keepdim=True)), v)
    return [out]


# ------------------------------------------------------------------------------------ work
def work(case):
    c, op = case, case["op"]
    if op == "rope":
        values = c["rows"] * (c["hq"] + c["hk"]) * c["d"]
        return {"bytes": 2 * SIZE[c["dtype"]] * values + 4 * len(_sections(c)) * c["rows"], "flops": 3 * c["rows"] * (c["hq"] + c["hk"]) * c["rot"]}
    if op == "norm":
        vectors = -(-c["rows"] // c["each"]) * (c["gate"] + 2 * c["mod"])
        return {"bytes": SIZE[c["dtype"]] * c["dim"] * (4 * c["rows"] + vectors) + 4 * c["dim"] * ((c["post"] != "none") + 1 + c["bias"]), "flops": 14 * c["rows"] * c["dim"]}
    if op == "pages":
        new = _lengths(c["new_lo"], c["new_hi"], c["b"], 2)
        # lengths in and sums out; a new block's entry and the list's, both ways; a row's position and slot
        return {"bytes": 20 * c["b"] + 16 * (sum(new) // c["page"] + 1) + 12 * sum(new), "flops": 4 * c["b"] + 4 * sum(new)}
    sizes, pre, tails = _sizes(c), _prefixes(c), _tails(c)
    tokens = sum(pre) + sum(tails)
    pairs = sum(n * p for n, p in zip(sizes, pre)) + sum(tails)
    return {"bytes": 2 * c["hkv"] * c["d"] * tokens + 8 * c["hkv"] * tokens // c["page"] + 2 * SIZE[c["dtype"]] * sum(sizes) * c["t"] * c["hq"] * c["d"],
            "flops": 4 * c["hq"] * c["d"] * c["t"] * pairs}
