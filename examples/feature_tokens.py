"""From a convolution's feature maps to decode steps over a cache, all on the GPU through the C ABI.

Two images' features go through a 3x3 convolution, a group norm with SiLU that leaves one row of channels
per pixel, and a 1x1 convolution that makes query, key and value rows of them (a [rows, C] matrix is an
NC4HW4 tensor of `rows` images of one pixel). The pixels attend to each other, image by image; their keys
and values go into the 8-bit cache; then each image's sequence takes a few steps of one token: project,
append, attend over the cache, project back.

    python examples/feature_tokens.py

prints how far the last step's rows are from the same chain in float64 with an exact cache.
"""
import ctypes
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import vknn_amd as V  # noqa: E402
from vknn_amd import DeviceBuffer, check  # noqa: E402

IMAGES, CIN, C, SIDE = 2, 96, 128, 14
Q_HEADS, KV_HEADS, DIM, PAGE, STEPS = 4, 2, 32, 64, 4
GROUPS, EPS, SCALE = 32, 1e-5, DIM ** -0.5
QKV = (Q_HEADS + 2 * KV_HEADS) * DIM
R = ctypes.byref


class Conv:
    """A stride-1 convolution with same padding, planned and packed once."""

    def __init__(self, n, cin, side, w):
        lib, k = V.vkhip(), w.shape[2]
        self.desc = V.ConvDesc(N=n, Cin=cin, H=side, W=side, Cout=w.shape[0], OH=side, OW=side, KH=k, KW=k, SH=1, SW=1, PT=k // 2, PL=k // 2, DH=1, DW=1, group=1)
        self.plan = V.ConvPlan()
        check(lib.vkhip_conv_plan_make(R(self.desc), V.CONV_AUTO, -1, 0, R(self.plan)), "conv plan")
        blob = np.zeros(self.plan.weight_bytes, np.uint8)
        w = np.ascontiguousarray(w, np.float32)
        check(lib.vkhip_conv_pack_weights(R(self.desc), R(self.plan), w.ctypes.data, None, blob.ctypes.data), "conv weights")
        self.blob, self.ws = DeviceBuffer.from_array(blob), DeviceBuffer(max(16, self.plan.workspace_bytes))
        self.ws.zero()
        self.out = DeviceBuffer(V.nc4_elems(n, w.shape[0], side, side) * 2)

    def __call__(self, x):
        check(V.vkhip().vkhip_conv_forward(R(self.desc), R(self.plan), x, self.blob.ptr, None, self.out.ptr, self.ws.ptr, None), "conv")
        return self.out.ptr


def ints(a):
    return DeviceBuffer.from_array(np.asarray(a, np.int32))


def half(a):
    return a.astype(np.float16).astype(np.float32)


def weights(rng):
    def normal(*shape):
        return half(rng.standard_normal(shape) * np.prod(shape[1:]) ** -0.5)
    return dict(conv=normal(C, CIN, 3, 3), qkv=normal(QKV, C, 1, 1), out=normal(C, Q_HEADS * DIM, 1, 1), gamma=rng.uniform(0.5, 1.5, C).astype(np.float32),
                beta=(rng.standard_normal(C) * 0.2).astype(np.float32))


def on_gpu(x, first, w):
    """x: feature maps NCHW, first: the first token's rows [IMAGES, C]. Returns the image attention's rows and the
    last step's."""
    lib = V.require_gpu()
    pixels = SIDE * SIDE
    rows = IMAGES * pixels
    packed, xf = DeviceBuffer(V.nc4_elems(IMAGES, CIN, SIDE, SIDE) * 2), DeviceBuffer.from_array(x)
    check(lib.vkhip_pack_nchw_f32(xf.ptr, packed.ptr, IMAGES, CIN, SIDE, SIDE, None), "pack")
    conv, qkv, qkv_step, out_step = Conv(IMAGES, CIN, SIDE, w["conv"]), Conv(rows, C, 1, w["qkv"]), Conv(IMAGES, C, 1, w["qkv"]), Conv(IMAGES, Q_HEADS * DIM, 1, w["out"])

    # feature map -> rows of channels
    gn = V.GroupNormDesc(N=IMAGES, C=C, H=SIDE, W=SIDE, groups=GROUPS, x_fmt=2, y_fmt=1, dtype=V.DT_F16, act=V.ACT["silu"], eps=EPS)
    gamma, beta, tokens = DeviceBuffer.from_array(w["gamma"]), DeviceBuffer.from_array(w["beta"]), DeviceBuffer(rows * C * 2)
    gn_ws = DeviceBuffer(lib.vkhip_group_norm_workspace_bytes(R(gn)))
    check(lib.vkhip_group_norm(R(gn), conv(packed.ptr), gamma.ptr, beta.ptr, tokens.ptr, gn_ws.ptr, None), "group_norm")
    q = qkv(tokens.ptr)
    k, v = q + Q_HEADS * DIM * 2, q + (Q_HEADS + KV_HEADS) * DIM * 2  # slices of the same rows

    # every pixel over its own image
    cu, att = ints([i * pixels for i in range(IMAGES + 1)]), DeviceBuffer(rows * Q_HEADS * DIM * 2)
    ad = V.AttentionDesc(batch=IMAGES, q_heads=Q_HEADS, kv_heads=KV_HEADS, head_dim=DIM, total_q=rows, total_k=rows, dtype=V.DT_F16, causal=0, scale=SCALE, q_row=QKV, q_head=DIM,
                         k_row=QKV, k_head=DIM, v_row=QKV, v_head=DIM, o_row=Q_HEADS * DIM, o_head=DIM)
    at_ws = DeviceBuffer(lib.vkhip_attention_workspace_bytes(R(ad)))
    check(lib.vkhip_attention_packed(R(ad), q, k, v, cu.ptr, cu.ptr, att.ptr, at_ws.ptr, None), "attention_packed")

    # the pixels' keys and values into the cache
    blocks = -(-(pixels + STEPS) // PAGE)
    pages, dp = IMAGES * blocks, lib.vkhip_kv_row(DIM)
    kp, vp = (DeviceBuffer(pages * KV_HEADS * PAGE * dp) for _ in range(2))
    ks, vs = (DeviceBuffer(pages * KV_HEADS * 4) for _ in range(2))
    table = ints(np.arange(pages).reshape(IMAGES, blocks)[:, ::-1])  # any pages in any order
    cache = V.KvCache(k=kp.ptr, v=vp.ptr, k_scale=ks.ptr, v_scale=vs.ptr, table=table.ptr, pages=pages, page_tokens=PAGE, kv_heads=KV_HEADS, head_dim=DIM, batch=IMAGES, max_blocks=blocks)
    strides = dict(dtype=V.DT_F16, k_row=QKV, k_head=DIM, v_row=QKV, v_head=DIM)
    empty = ints([0] * IMAGES)
    check(lib.vkhip_kv_append(R(cache), R(V.KvRows(total=rows, **strides)), k, v, cu.ptr, empty.ptr, None), "kv_append")

    # steps of one token per image
    kd = V.KvAttentionDesc(q_heads=Q_HEADS, q_tokens=1, dtype=V.DT_F16, max_len=pixels + STEPS, scale=SCALE, q_row=QKV, q_head=DIM, o_row=Q_HEADS * DIM, o_head=DIM)
    kd_ws, seen, one = DeviceBuffer(lib.vkhip_kv_attention_workspace_bytes(R(kd), R(cache))), DeviceBuffer(IMAGES * Q_HEADS * DIM * 2), ints(range(IMAGES + 1))
    row = DeviceBuffer.from_array(first.astype(np.float16))
    x_step = row.ptr
    for i in range(STEPS):
        before, now = ints([pixels + i] * IMAGES), ints([pixels + i + 1] * IMAGES)
        q = qkv_step(x_step)
        k, v = q + Q_HEADS * DIM * 2, q + (Q_HEADS + KV_HEADS) * DIM * 2
        check(lib.vkhip_kv_append(R(cache), R(V.KvRows(total=IMAGES, **strides)), k, v, one.ptr, before.ptr, None), "kv_append")
        check(lib.vkhip_kv_attention(R(kd), R(cache), q, now.ptr, seen.ptr, kd_ws.ptr, None), "kv_attention")
        x_step = out_step(seen.ptr)
        check(lib.vkhip_stream_sync(None), "sync")  # `before` and `now` are freed
    return att.download(np.float16, rows * Q_HEADS * DIM).astype(np.float64).reshape(rows, -1), out_step.out.download(np.float16, IMAGES * C).astype(np.float64).reshape(IMAGES, C)


def softmax_attention(q, k, v):
    """q [n, Q_HEADS, DIM], k, v [m, KV_HEADS, DIM]"""
    o = np.empty(q.shape)
    for h in range(Q_HEADS):
        kv = h * KV_HEADS // Q_HEADS
        z = q[:, h] @ k[:, kv].T * SCALE
        p = np.exp(z - z.max(1, keepdims=True))
        o[:, h] = p / p.sum(1, keepdims=True) @ v[:, kv]
    return o


def in_float64(x, first, w):
    x, pixels = x.astype(np.float64), SIDE * SIDE
    xp = np.pad(x, ((0, 0), (0, 0), (1, 1), (1, 1)))
    y = sum(np.einsum("oc,nchw->nohw", w["conv"][:, :, i, j].astype(np.float64), xp[:, :, i:i + SIDE, j:j + SIDE]) for i in range(3) for j in range(3))
    t = y.reshape(IMAGES, C, pixels).transpose(0, 2, 1).reshape(IMAGES, pixels, GROUPS, C // GROUPS)
    t = (t - t.mean((1, 3), keepdims=True)) / np.sqrt(t.var((1, 3), keepdims=True) + EPS)
    t = t.reshape(IMAGES, pixels, C) * w["gamma"] + w["beta"]
    t = t / (1 + np.exp(-t))
    qkv, out = w["qkv"][:, :, 0, 0].astype(np.float64), w["out"][:, :, 0, 0].astype(np.float64)

    def project(rows):
        r = (rows @ qkv.T).reshape(len(rows), -1, DIM)
        return r[:, :Q_HEADS], r[:, Q_HEADS:Q_HEADS + KV_HEADS], r[:, Q_HEADS + KV_HEADS:]

    att, last = [], []
    for i in range(IMAGES):
        q, k, v = project(t[i])
        att.append(softmax_attention(q, k, v).reshape(pixels, -1))
        row = first[i:i + 1].astype(np.float64)
        for _ in range(STEPS):
            q, k1, v1 = project(row)
            k, v = np.concatenate([k, k1]), np.concatenate([v, v1])
            row = softmax_attention(q, k, v).reshape(1, -1) @ out.T
        last.append(row)
    return np.concatenate(att), np.concatenate(last)


def main():
    rng = np.random.default_rng(3)
    w = weights(rng)
    x, first = half(rng.standard_normal((IMAGES, CIN, SIDE, SIDE))), half(rng.standard_normal((IMAGES, C)))
    errors = []
    for name, got, want in zip(("attention rows", "last step"), on_gpu(x, first, w), in_float64(x, first, w)):
        errors.append(np.linalg.norm(got - want) / np.linalg.norm(want))
        print("%s: relative error %.2e" % (name, errors[-1]))
    return errors


if __name__ == "__main__":
    main()
