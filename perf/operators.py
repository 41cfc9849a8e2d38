"""What leads from this framework's feature maps to token models, as cases that can be timed and checked:
group norm with an activation to channels-last rows, attention over packed sequences, rows into and out
of an 8-bit cache of pages, and attention over that cache. Each case is one call (or the pair of calls
that belong together) of the kernel library's C ABI (include/vkhip.h) on tensors that sit on the GPU, on
the program's current stream; the plain forms are the same operators in elementary float32 tensor
operations.
"""
import ctypes
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
DT_CODE = {"f16": 0, "bf16": 1, "f32": 2}
ACT = {"none": 0, "relu": 1, "hardswish": 4, "silu": 5}
FMT = {"nhwc": 1, "nc4": 2}
EPS = 1e-5


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One image's 40 x 40 level of a detector neck (YOLOv8n's 128 channels): a call of a few microseconds.
        dict(name="gn_b1", op="gn", n=1, c=128, h=40, w=40, groups=32, x="nhwc", y="nhwc", dtype="f16", act="silu"),
        # An odd map (600 x 600 images at stride 8) with 108 channels, from the convolutions' NC4HW4 to rows of channels.
        dict(name="gn_odd_b8", op="gn", n=8, c=108, h=75, w=75, groups=27, x="nc4", y="nhwc", dtype="f16", act="silu"),
        # A large batch of ResNet-50's second stage, the largest map that gets a norm: 205 MB in and out.
        dict(name="gn_b64", op="gn", n=64, c=256, h=56, w=56, groups=32, x="nhwc", y="nhwc", dtype="f16", act="relu"),
        # Four images of different sizes as tokens of the 7 x 7 to 14 x 14 maps, all keys visible: a few microseconds.
        dict(name="attn_images", op="attn", b=4, lo=49, hi=196, prefix=0, hq=8, hkv=8, d=64, causal=False, dtype="f16"),
        # A batch of prompts of different lengths with grouped heads: ordinary work of a decoder.
        dict(name="attn_prompts", op="attn", b=8, lo=300, hi=4000, prefix=0, hq=32, hkv=8, d=128, causal=True, dtype="bf16"),
        # One long prompt: where the matrix units count.
        dict(name="attn_long", op="attn", b=1, lo=16384, hi=16384, prefix=0, hq=32, hkv=8, d=128, causal=True, dtype="f16"),
        # A decode step's new token for 64 sequences into their pages, and the page that holds it back as rows.
        dict(name="rows_step", op="rows", b=64, new_lo=1, new_hi=1, old_lo=1, old_hi=1000, hkv=8, d=128, page=64, back="page", dtype="f16"),
        # Chunks of prompts behind cached prefixes, and the whole sequences back as rows for the chunks' attention.
        dict(name="rows_prompt", op="rows", b=8, new_lo=300, new_hi=4000, old_lo=0, old_hi=700, hkv=8, d=128, page=64, back="all", dtype="bf16"),
        # One sequence, one token: latency.
        dict(name="step_b1", op="step", b=1, lo=1000, hi=1000, t=1, hq=32, hkv=8, d=128, page=64, dtype="f16"),
        # The ordinary decode step: 64 sequences of different lengths.
        dict(name="step_b64", op="step", b=64, lo=200, hi=4000, t=1, hq=32, hkv=8, d=128, page=64, dtype="f16"),
        # Five drafted tokens per sequence with smaller heads and pages.
        dict(name="step_draft", op="step", b=16, lo=500, hi=9000, t=5, hq=16, hkv=4, d=64, page=32, dtype="bf16"),
        # A few very long sequences: the largest cache, more than 2^31 bytes of pages.
        dict(name="step_long", op="step", b=8, lo=100000, hi=160000, t=1, hq=32, hkv=8, d=128, page=64, dtype="f16"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = {k: max(work(c)["bytes" if k != "attn" else "flops"] for c in listed() if c["op"] == k) for k in ("gn", "attn", "rows", "step")}
    op = rng.choice(["gn", "gn", "attn", "attn", "attn", "rows", "rows", "step", "step", "step"])
    while True:
        dtype = rng.choice(["f16", "bf16"])
        if op == "gn":
            # maps of 7 to 112 pixels a side, 16 to 512 channels, batch 1 to 64; float32 rows too
            c = _log(rng, 16, 512) // 4 * 4
            groups = rng.choice([g for g in range(1, c + 1) if c % g == 0 and c // g >= 2 and g <= 64])
            x, y = rng.choice([("nhwc", "nhwc"), ("nc4", "nhwc"), ("nc4", "nc4"), ("nhwc", "nc4")])
            case = dict(op=op, n=_log(rng, 1, 64), c=c, h=_log(rng, 7, 112), w=_log(rng, 7, 112), groups=groups, x=x, y=y,
                        dtype=rng.choice(["f16", "f16", "bf16", "f32"]) if x == y == "nhwc" else "f16", act=rng.choice(["none", "relu", "hardswish", "silu"]))
        elif op == "attn":
            # 1 to 16 sequences of 1 to 16384 tokens, behind no prefix or one; heads of 32 to 128
            hi = _log(rng, 40, 16384)
            hkv = rng.choice([1, 2, 4, 8])
            case = dict(op=op, b=_log(rng, 1, 16), lo=rng.randint(1, hi), hi=hi, prefix=rng.choice([0, 0, _log(rng, 1, 2000)]), hq=hkv * rng.choice([1, 2, 4, 6]), hkv=hkv,
                        d=rng.choice([32, 64, 80, 96, 128, 128]), causal=rng.random() < 0.7, dtype=dtype)
        elif op == "rows":
            new = rng.choice([1, 1, _log(rng, 2, 4000)])
            case = dict(op=op, b=_log(rng, 1, 64), new_lo=rng.randint(1, new), new_hi=new, old_lo=0, old_hi=_log(rng, 1, 2000), hkv=rng.choice([1, 2, 4, 8]),
                        d=rng.choice([64, 96, 128]), page=rng.choice([32, 64, 128]), back=rng.choice(["page", "all"]), dtype=dtype)
        else:
            hi = _log(rng, 20, 160000)
            hkv = rng.choice([1, 2, 4, 8])
            case = dict(op=op, b=_log(rng, 1, 64), lo=max(1, int(hi * rng.random())), hi=hi, t=rng.choice([1, 1, 1, 2, 5, 8]), hq=hkv * rng.choice([1, 2, 4, 8]), hkv=hkv,
                        d=rng.choice([64, 96, 128]), page=rng.choice([32, 64, 128]), dtype=dtype)
        w = work(case)
        if w["bytes" if op != "attn" else "flops"] <= most[op] and w["bytes"] <= 3e9:
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


def _cu(lens):
    return [0] + [int(v) for v in np.cumsum(lens)]


def _dp(d):
    return 64 if d <= 64 else 128


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 131 + salt) & 0x7FFFFFFF)
    return g


def _ints(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _seqs(c):
    """(queries, keys) of each sequence of an attention case."""
    q = _lengths(c["lo"], c["hi"], c["b"], 1)
    return q, [n + c["prefix"] for n in q]


def _pages(c, lens, seed):
    """A cache whose sequences hold `lens` tokens: page table (pages in a mixed order), int8 pages, scales."""
    page, hkv, d, dp, b = c["page"], c["hkv"], c["d"], _dp(c["d"]), c["b"]
    blocks = [-(-n // page) for n in lens]
    width, total = max(blocks), sum(blocks) + 1
    order = np.random.default_rng([seed & 0x7FFFFFFF, 5]).permutation(total)[:sum(blocks)]
    table = np.full((b, width), -1, np.int32)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
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
    return dict(k=k, v=v, ks=ks, vs=vs, table=torch.from_numpy(table).cuda(), pages=total, width=width)


def _inputs(c, seed):
    """Everything random of a case."""
    dt, op = DTYPES[c["dtype"]], c["op"]
    if op == "gn":
        n, ch, h, w = c["n"], c["c"], c["h"], c["w"]
        # what a convolution leaves: channels of different means and deviations
        g = _gen(seed, 1)
        x = torch.randn((n, h * w, ch), generator=g, device="cuda")
        x = x * (torch.rand(ch, generator=g, device="cuda") + 0.5) + torch.randn(ch, generator=g, device="cuda")
        x = x.to(dt)
        if c["x"] == "nc4":
            x = x.view(n, h * w, ch // 4, 4).permute(0, 2, 1, 3).contiguous()
        return dict(x=x, gamma=torch.rand(ch, generator=g, device="cuda") + 0.5, beta=torch.randn(ch, generator=g, device="cuda") * 0.2)
    if op == "attn":
        nq, nk = _seqs(c)
        g = _gen(seed, 2)
        # one product of a projection makes query, key and value rows side by side where nothing is cached
        hq, hkv, d = c["hq"], c["hkv"], c["d"]
        if c["prefix"] == 0:
            qkv = torch.randn((sum(nq), (hq + 2 * hkv) * d), generator=g, device="cuda").to(dt)
            q, k, v = qkv[:, :hq * d], qkv[:, hq * d:(hq + hkv) * d], qkv[:, (hq + hkv) * d:]
        else:
            q = torch.randn((sum(nq), hq * d), generator=g, device="cuda").to(dt)
            k, v = (torch.randn((sum(nk), hkv * d), generator=g, device="cuda").to(dt) for _ in range(2))
        return dict(q=q.unflatten(1, (hq, d)), k=k.unflatten(1, (hkv, d)), v=v.unflatten(1, (hkv, d)), nq=nq, nk=nk)
    if op == "rows":
        old = _lengths(c["old_lo"], c["old_hi"], c["b"], 2)
        new = _lengths(c["new_lo"], c["new_hi"], c["b"], 3)
        p = _pages(c, [o + n for o, n in zip(old, new)], seed)
        g = _gen(seed, 4)
        k, v = (torch.randn((sum(new), c["hkv"], c["d"]), generator=g, device="cuda").to(dt) for _ in range(2))
        first = [o // c["page"] * c["page"] if c["back"] == "page" else 0 for o in old]
        return dict(p, new_k=k, new_v=v, old=old, new=new, first=first)
    lens = _lengths(c["lo"], c["hi"], c["b"], 4)
    q = torch.randn((c["b"], c["t"], c["hq"], c["d"]), generator=_gen(seed, 6), device="cuda").to(dt)
    return dict(_pages(c, lens, seed), q=q, lens=lens)


# ------------------------------------------------------------------------------------ state and passes
def prepare(case, seed):
    c, d = dict(case), _inputs(case, seed)
    dt, op = DTYPES[c["dtype"]], c["op"]
    st = {"case": c, **d}
    if op == "gn":
        n, hw = c["n"], c["h"] * c["w"]
        st["out"] = torch.empty((n, hw, c["c"]) if c["y"] == "nhwc" else (n, c["c"] // 4, hw, 4), dtype=dt, device="cuda")
    elif op == "attn":
        st.update(cu_q=_ints(_cu(d["nq"])), cu_k=_ints(_cu(d["nk"])), out=torch.empty((sum(d["nq"]), c["hq"], c["d"]), dtype=dt, device="cuda"))
    elif op == "rows":
        back = [o + n - f for o, n, f in zip(d["old"], d["new"], d["first"])]
        st.update(back=back, cu_new=_ints(_cu(d["new"])), lens=_ints(d["old"]), cu_back=_ints(_cu(back)), start=_ints(d["first"]),
                  out_k=torch.empty((sum(back), c["hkv"], c["d"]), dtype=dt, device="cuda"), out_v=torch.empty((sum(back), c["hkv"], c["d"]), dtype=dt, device="cuda"))
    else:
        st.update(lens_gpu=_ints(d["lens"]), out=torch.empty_like(d["q"]))
    if own:
        _prepare_own(st)
    torch.cuda.synchronize()
    return st


def _prepare_own(st):
    """The descriptors and the workspace that a program keeps beside its tensors."""
    import vknn_amd as V
    lib, c, op = V.require_gpu(), st["case"], st["case"]["op"]
    st.update(lib=lib, check=V.check)
    code = DT_CODE[c["dtype"]]
    ws = 0
    if op == "gn":
        st["desc"] = V.GroupNormDesc(N=c["n"], C=c["c"], H=c["h"], W=c["w"], groups=c["groups"], x_fmt=FMT[c["x"]], y_fmt=FMT[c["y"]], dtype=code,
                                     act=ACT[c["act"]], act_lo=0.0, act_hi=0.0, eps=EPS, x_row=0, y_row=0)
        ws = lib.vkhip_group_norm_workspace_bytes(ctypes.byref(st["desc"]))
    elif op == "attn":
        q, k, v, o = st["q"], st["k"], st["v"], st["out"]
        st["desc"] = V.AttentionDesc(batch=c["b"], q_heads=c["hq"], kv_heads=c["hkv"], head_dim=c["d"], total_q=q.shape[0], total_k=k.shape[0], dtype=code,
                                     causal=int(c["causal"]), scale=c["d"] ** -0.5, q_row=q.stride(0), q_head=q.stride(1), k_row=k.stride(0), k_head=k.stride(1),
                                     v_row=v.stride(0), v_head=v.stride(1), o_row=o.stride(0), o_head=o.stride(1))
        ws = lib.vkhip_attention_workspace_bytes(ctypes.byref(st["desc"]))
    else:
        st["cache"] = V.KvCache(k=st["k"].data_ptr(), v=st["v"].data_ptr(), k_scale=st["ks"].data_ptr(), v_scale=st["vs"].data_ptr(), table=st["table"].data_ptr(),
                                pages=st["pages"], page_tokens=c["page"], kv_heads=c["hkv"], head_dim=c["d"], batch=c["b"], max_blocks=st["width"])
        if op == "rows":
            row = dict(dtype=code, k_row=c["hkv"] * c["d"], k_head=c["d"], v_row=c["hkv"] * c["d"], v_head=c["d"])
            st.update(rows_new=V.KvRows(total=st["new_k"].shape[0], **row), rows_back=V.KvRows(total=st["out_k"].shape[0], **row))
        else:
            q = st["q"]
            st["desc"] = V.KvAttentionDesc(q_heads=c["hq"], q_tokens=c["t"], dtype=code, max_len=max(st["lens"]), scale=c["d"] ** -0.5,
                                           q_row=q.stride(1), q_head=q.stride(2), o_row=q.stride(1), o_head=q.stride(2))
            ws = lib.vkhip_kv_attention_workspace_bytes(ctypes.byref(st["desc"]), ctypes.byref(st["cache"]))
    st["ws"] = torch.empty(max(ws, 16), dtype=torch.uint8, device="cuda")


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(st):
    lib, op, ref = st["lib"], st["case"]["op"], ctypes.byref
    # the library's NULL is its own stream; 1 is the runtime's handle of the default stream
    s = torch.cuda.current_stream().cuda_stream or 1
    if op == "gn":
        st["check"](lib.vkhip_group_norm(ref(st["desc"]), st["x"].data_ptr(), st["gamma"].data_ptr(), st["beta"].data_ptr(), st["out"].data_ptr(),
                                         st["ws"].data_ptr(), s), "group_norm")
        return [st["out"]]
    if op == "attn":
        st["check"](lib.vkhip_attention_packed(ref(st["desc"]), st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["cu_q"].data_ptr(),
                                               st["cu_k"].data_ptr(), st["out"].data_ptr(), st["ws"].data_ptr(), s), "attention_packed")
        return [st["out"]]
    if op == "rows":
        st["check"](lib.vkhip_kv_append(ref(st["cache"]), ref(st["rows_new"]), st["new_k"].data_ptr(), st["new_v"].data_ptr(), st["cu_new"].data_ptr(),
                                        st["lens"].data_ptr(), s), "kv_append")
        st["check"](lib.vkhip_kv_read(ref(st["cache"]), ref(st["rows_back"]), st["start"].data_ptr(), st["cu_back"].data_ptr(), st["out_k"].data_ptr(),
                                      st["out_v"].data_ptr(), s), "kv_read")
        return [st["out_k"], st["out_v"], st["ks"], st["vs"]]
    st["check"](lib.vkhip_kv_attention(ref(st["desc"]), ref(st["cache"]), st["q"].data_ptr(), st["lens_gpu"].data_ptr(), st["out"].data_ptr(),
                                       st["ws"].data_ptr(), s), "kv_attention")
    return [st["out"]]


def _act(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "hardswish":
        return v * (v + 3).clamp(0, 6) / 6
    return v / (1 + torch.exp(-v)) if act == "silu" else v


def _softmax_rows(s):
    """exp(s - max) / sum over the last axis; a row of -inf alone gives zeros."""
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0, m))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _run_plain(st):
    c, op = st["case"], st["case"]["op"]
    dt = DTYPES[c["dtype"]]
    if op == "gn":
        n, ch, hw, g = c["n"], c["c"], c["h"] * c["w"], c["groups"]
        x = st["x"].float()
        if c["x"] == "nc4":
            x = x.permute(0, 2, 1, 3).reshape(n, hw, ch)
        x = x.view(n, hw, g, ch // g)
        mean = x.mean((1, 3), keepdim=True)
        x = x - mean
        rstd = torch.rsqrt((x * x).mean((1, 3), keepdim=True) + EPS)
        y = _act((x * rstd).view(n, hw, ch) * st["gamma"] + st["beta"], c["act"]).to(dt)
        return [y.view(n, hw, ch // 4, 4).permute(0, 2, 1, 3).contiguous() if c["y"] == "nc4" else y]
    if op == "attn":
        hq, hkv, d = c["hq"], c["hkv"], c["d"]
        out = torch.empty((sum(st["nq"]), hq, d), dtype=dt, device="cuda")
        q0 = k0 = 0
        for nq, nk in zip(st["nq"], st["nk"]):
            step = max(1, min(nq, (1 << 28) // max(1, nk * hq)))  # rows at a time, so that their scores fit
            k = st["k"][k0:k0 + nk].float().permute(1, 2, 0).contiguous()
            v = st["v"][k0:k0 + nk].float().transpose(0, 1).contiguous()
            for i in range(0, nq, step):
                e = min(nq, i + step)
                see = e + nk - nq if c["causal"] else nk
                q = st["q"][q0 + i:q0 + e].float().transpose(0, 1).reshape(hkv, hq // hkv * (e - i), d)
                s = torch.matmul(q, k[:, :, :see]).view(hq, e - i, see) * d ** -0.5
                if c["causal"]:
                    at = torch.arange(i, e, device="cuda") + (nk - nq)
                    s.masked_fill_(torch.arange(see, device="cuda") > at[:, None], -math.inf)
                o = torch.matmul(_softmax_rows(s).view(hkv, -1, see), v[:, :see])
                out[q0 + i:q0 + e] = o.view(hq, e - i, d).transpose(0, 1).to(dt)
            q0 += nq
            k0 += nk
        return [out]
    table = st["table"]
    page, hkv, d = c["page"], c["hkv"], c["d"]
    if op == "rows":
        at = 0
        outs_k, outs_v = [], []
        for i, (old, new, first) in enumerate(zip(st["old"], st["new"], st["first"])):
            k, v = st["new_k"][at:at + new].float(), st["new_v"][at:at + new].float()
            at += new
            # the first page may hold tokens already: its scale grows and they are rounded again
            b0, b1 = old // page, -(-(old + new) // page)
            ids = table[i, b0:b1].long()
            have = old - b0 * page
            for x, pool, scale, by_token in ((k, st["k"], st["ks"], True), (v, st["v"], st["vs"], False)):
                full = torch.zeros(((b1 - b0) * page, hkv, d), device="cuda")
                full[have:have + new] = x
                full = full.view(b1 - b0, page, hkv, d).permute(0, 2, 1, 3)  # page, head, token, channel
                before = torch.zeros((b1 - b0, hkv), device="cuda")
                if have:
                    before[0] = scale[ids[0]]
                s = torch.maximum(before, full.abs().amax((2, 3)) / 127)
                safe = torch.where(s > 0, s, 1)[:, :, None, None]
                qs = torch.round(full / safe).clamp(-127, 127)
                if have:
                    was = pool[ids[0]] if by_token else pool[ids[0]].transpose(1, 2)
                    qs[0, :, :have] = torch.round(was[:, :have, :d].float() * (before[0] / safe[0, :, 0, 0])[:, None, None])
                cells = pool[ids] if by_token else pool[ids].transpose(2, 3)
                tok = torch.arange((b1 - b0) * page, device="cuda").view(b1 - b0, 1, page, 1)
                cells[..., :d] = torch.where(tok < have + new, qs, cells[..., :d].float()).to(torch.int8)
                pool[ids] = cells if by_token else cells.transpose(2, 3)
                scale[ids] = s
            f0 = first // page
            rd = table[i, f0:b1].long()
            rk = (st["k"][rd][..., :d].float() * st["ks"][rd][:, :, None, None]).permute(0, 2, 1, 3).reshape(-1, hkv, d)
            rv = (st["v"][rd][:, :, :d].float() * st["vs"][rd][:, :, None, None]).permute(0, 3, 1, 2).reshape(-1, hkv, d)
            outs_k.append(rk[first - f0 * page:old + new - f0 * page].to(dt))
            outs_v.append(rv[first - f0 * page:old + new - f0 * page].to(dt))
        return [torch.cat(outs_k), torch.cat(outs_v), st["ks"], st["vs"]]
    t, hq = c["t"], c["hq"]
    out = torch.empty_like(st["q"])
    for i, n in enumerate(st["lens"]):
        ids = table[i, :-(-n // page)].long()
        k = (st["k"][ids][..., :d].float() * st["ks"][ids][:, :, None, None]).permute(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n]
        v = (st["v"][ids][:, :, :d].float() * st["vs"][ids][:, :, None, None]).permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :n]
        q = st["q"][i].float().transpose(0, 1).reshape(hkv, hq // hkv * t, d)
        s = (torch.matmul(q, k.transpose(1, 2)) * d ** -0.5).view(hq, t, n)
        if t > 1:
            s.masked_fill_(torch.arange(n, device="cuda") > (torch.arange(t, device="cuda") + (n - t))[:, None], -math.inf)
        out[i] = torch.matmul(_softmax_rows(s).view(hkv, -1, n), v).view(hq, t, d).transpose(0, 1).to(out.dtype)
    return [out]


# ------------------------------------------------------------------------------------ float64 values
def exact(case, seed):
    c, d, op = case, _inputs(case, seed), case["op"]
    if op == "gn":
        n, ch, hw, g = c["n"], c["c"], c["h"] * c["w"], c["groups"]
        x = d["x"].double()
        if c["x"] == "nc4":
            x = torch.cat([x[:, i] for i in range(ch // 4)], 2)
        y = torch.empty_like(x)
        for i in range(g):
            cols = slice(i * (ch // g), (i + 1) * (ch // g))
            part = x[:, :, cols]
            var, mean = torch.var_mean(part, dim=(1, 2), keepdim=True, correction=0)
            y[:, :, cols] = (part - mean) / (var + EPS).sqrt() * d["gamma"].double()[cols] + d["beta"].double()[cols]
        if c["act"] == "relu":
            y.clamp_(min=0)
        elif c["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif c["act"] == "hardswish":
            y = y * ((y + 3) / 6).clamp(0, 1)
        return [torch.stack([y[:, :, i:i + 4] for i in range(0, ch, 4)], 1) if c["y"] == "nc4" else y]
    if op == "attn":
        group, dim = c["hq"] // c["hkv"], c["d"]
        out = torch.zeros((sum(d["nq"]), c["hq"], dim), dtype=torch.float64, device="cuda")
        cq, ck = _cu(d["nq"]), _cu(d["nk"])
        for b in range(c["b"]):
            nq, nk = d["nq"][b], d["nk"][b]
            for h in range(c["hq"]):
                k = d["k"][ck[b]:ck[b + 1], h // group].double()
                v = d["v"][ck[b]:ck[b + 1], h // group].double()
                for i in range(0, nq, 4096):
                    rows = torch.arange(i, min(nq, i + 4096), device="cuda")
                    z = d["q"][cq[b] + i:cq[b] + i + len(rows), h].double() @ k.t() / math.sqrt(dim)
                    if c["causal"]:
                        z = torch.where(torch.arange(nk, device="cuda")[None] <= rows[:, None] + nk - nq, z, -math.inf)
                    out[cq[b] + i:cq[b] + i + len(rows), h] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ v
        return [out]
    page, dim, hkv = c["page"], c["d"], c["hkv"]
    table = d["table"].cpu().numpy()
    if op == "rows":
        scales = [d["ks"].double(), d["vs"].double()]
        outs = [[], []]
        at = 0
        for b in range(c["b"]):
            old, new, first = d["old"][b], d["new"][b], d["first"][b]
            for which in range(2):
                x = (d["new_k"], d["new_v"])[which][at:at + new].double()
                pool = (d["k"], d["v"])[which]
                values = []
                for blk in range(first // page, -(-(old + new) // page)):
                    pid, lo, hi = int(table[b, blk]), blk * page, min(old + new, (blk + 1) * page)
                    held = pool[pid].double() if which == 0 else pool[pid].double().transpose(1, 2)
                    held = held[:, :, :dim]
                    s0 = scales[which][pid].clone()
                    n0 = max(0, min(old, hi) - lo)
                    if n0 < hi - lo:
                        add = x[max(lo, old) - old:hi - old].transpose(0, 1)
                        s = add.abs().amax((1, 2)) / 127
                        if n0:
                            s = torch.maximum(s, s0)
                        div = torch.where(s > 0, s, 1)[:, None, None]
                        q = torch.round(add / div)
                        if n0:
                            q = torch.cat([torch.round(held[:, :n0] * s0[:, None, None] / div), q], 1)
                        scales[which][pid] = s
                    else:
                        q, s = held[:, :n0], s0
                    values.append((q * s[:, None, None]).transpose(0, 1)[max(0, first - lo):])
                outs[which] += values
            at += new
        return [torch.cat(outs[0]), torch.cat(outs[1])] + scales
    group, t = c["hq"] // hkv, c["t"]
    out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["b"]):
        n = d["lens"][b]
        ids = torch.from_numpy(table[b, :-(-n // page)].astype(np.int64)).cuda()
        for h in range(hkv):
            k = (d["k"][ids, h].double() * d["ks"][ids, h].double()[:, None, None]).flatten(0, 1)[:n, :dim]
            v = (d["v"][ids, h].double() * d["vs"][ids, h].double()[:, None, None]).transpose(1, 2).flatten(0, 1)[:n, :dim]
            for r in range(group):
                for i in range(t):
                    see = n - t + i + 1
                    if see <= 0:
                        continue
                    z = k[:see] @ d["q"][b, i, h * group + r].double() / math.sqrt(dim)
                    out[b, i, h * group + r] = torch.exp(z - torch.logsumexp(z, 0)) @ v[:see]
    return [out]


# ------------------------------------------------------------------------------------ work
def work(case):
    c, op = case, case["op"]
    size = 4 if c["dtype"] == "f32" else 2
    if op == "gn":
        n = c["n"] * c["c"] * c["h"] * c["w"]
        return {"bytes": 2 * size * n + 8 * c["c"], "flops": 10 * n}
    if op == "attn":
        nq, nk = _seqs(c)
        pairs = sum(q * (k - q) + q * (q + 1) // 2 if c["causal"] else q * k for q, k in zip(nq, nk))
        return {"bytes": size * c["d"] * (2 * c["hq"] * sum(nq) + 2 * c["hkv"] * sum(nk)), "flops": 4 * c["hq"] * c["d"] * pairs}
    if op == "rows":
        old, new = _lengths(c["old_lo"], c["old_hi"], c["b"], 2), _lengths(c["new_lo"], c["new_hi"], c["b"], 3)
        back = sum(o + n - (o // c["page"] * c["page"] if c["back"] == "page" else 0) for o, n in zip(old, new))
        row = 2 * c["hkv"] * c["d"]
        # new rows in and their bytes out; the bytes of what is read back, once, and its rows out
        return {"bytes": row * ((size + 1) * sum(new) + (size + 1) * back), "flops": row * (2 * sum(new) + back)}
    lens = _lengths(c["lo"], c["hi"], c["b"], 4)
    scales = 8 * c["hkv"] * sum(-(-n // c["page"]) for n in lens)
    return {"bytes": 2 * c["hkv"] * c["d"] * sum(lens) + scales + 2 * size * c["b"] * c["t"] * c["hq"] * c["d"],
            "flops": 4 * c["hq"] * c["d"] * c["t"] * sum(lens)}
