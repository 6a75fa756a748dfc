"""Layer norm, 8-bit activation checkpoints and cross attention on the GPU against their definitions in 64 bits (tests/token_ref.py, with its
element-by-element bounds), their refusals, streams, graphs, and the matching attention that the trainer builds from them."""
import contextlib
import random

import numpy as np
import pytest
import torch

import token_ref as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g) * scale + shift).to(dtype).cuda()


def check(got, want, what):
    for name, t in got.items():
        ref.within(t, want[name][0], want[name][1], "%s %s" % (what, name))


# --------------------------------------------------------------------------- 8-bit activations
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("n", [0, 1, 31, 32, 33, 255, 1024, 4099, 100003])
def test_act8_values(dtype, n):
    from movedepth_amd import ops

    g = gen(n)
    x = randn(g, n, dtype=DT[dtype], scale=1.0)
    x = (x.float() * torch.exp2(torch.randint(-9, 4, (n,), generator=g).float()).cuda()).to(DT[dtype])
    p = ops.act8_pack(x)
    back = ops.act8_unpack(p)
    assert back.dtype == x.dtype and back.shape == x.shape and p.nbytes() == n + (n + 31) // 32
    assert torch.equal(back.double().cpu(), ref.act8(x.view(1, -1))[0])
    again = ops.act8_pack(back)
    assert torch.equal(again.codes, p.codes) and torch.equal(again.scales, p.scales)


@pytest.mark.parametrize("dtype", DT)
def test_act8_ends_of_the_range(dtype):
    """zeros, the smallest and the largest values, the border between two steps, infinities and NaN"""
    from movedepth_amd import ops

    dt = DT[dtype]
    f = torch.finfo(dt)
    rows = [[0.0], [-0.0, 0.0], [f.smallest_normal], [f.smallest_normal * f.eps, -f.smallest_normal], [f.max], [-f.max, 1.0], [127.0, 1.0, 0.5],
            [127.25, 1.0], [127.5, 0.5, 1.5, 2.5], [128.0, 1.0], [255.0, 1.0, 3.0], [256.0], [1e-3, 1e-5], [f.max, f.max / 2, f.max / 300]]
    x = torch.zeros(len(rows), 32, dtype=torch.float64)
    for i, r in enumerate(rows):
        x[i, :len(r)] = torch.tensor(r, dtype=torch.float64)
    x = x.to(dt).cuda()
    back = ops.act8_unpack(ops.act8_pack(x))
    assert torch.equal(back.double().cpu(), ref.act8(x))
    assert bool(torch.isfinite(back).all())
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = torch.ones(96, dtype=dt, device="cuda")
        y[40] = bad
        z = ops.act8_unpack(ops.act8_pack(y))
        assert bool(torch.isnan(z[32:64]).all()) and torch.equal(z[:32], y[:32]) and torch.equal(z[64:], y[64:])


def test_act8_layouts():
    """storage order, strides and offsets come back; a view that does not fill its memory is packed as a copy"""
    from movedepth_amd import ops

    x = randn(gen(1), 2, 16, 3, 5, 7)
    for t in (x, x.contiguous(memory_format=torch.channels_last_3d), x.permute(3, 0, 4, 1, 2), x[1], x.flatten()[1:], x[:, ::2], x[:, :1].expand(2, 4, 3, 5, 7)):
        b = ops.act8_unpack(ops.act8_pack(t))
        assert b.shape == t.shape
        dense = t if ops._is_dense(t) else t.contiguous()
        assert b.stride() == dense.stride()
        flat = dense.as_strided((dense.numel(),), (1,), dense.storage_offset())
        assert torch.equal(b.as_strided((b.numel(),), (1,)).double().cpu(), ref.act8(flat.view(1, -1))[0])
    with pytest.raises(RuntimeError):
        ops.act8_pack(torch.zeros(4, dtype=torch.float64, device="cuda"))


def test_saved_act8_in_autograd():
    """what autograd keeps inside the context is the 8-bit value; outside, small tensors, and parameters stay as they are"""
    from movedepth_amd import ops

    g = gen(3)
    x, w, go = randn(g, 64, 100).requires_grad_(), randn(g, 64, 100).requires_grad_(), randn(g, 64, 100)
    a = x * 1.0
    with ops.saved_act8(min_numel=64 * 100):
        y = a * w                       # keeps a (an activation) and w (a leaf)
    gx, gw = torch.autograd.grad(y, (x, w), go)
    assert torch.equal(gx, go * w)
    a8 = ref.act8((x * 1.0).view(1, -1)).view(64, 100)
    ref.within(gw, go.double().cpu() * a8, 2.0 ** -24 * (go.double().cpu() * a8).abs(), "dw")
    with ops.saved_act8(min_numel=64 * 100 + 1):
        y = (x * 1.0) * w
    assert torch.equal(torch.autograd.grad(y, w, go)[0], go * x)


# --------------------------------------------------------------------------- layer norm
def run_layer_norm(x, w, b, eps, g, act_bits=0):
    from movedepth_amd import ops

    x = x.detach().requires_grad_()
    w, b = (None if t is None else t.detach().requires_grad_() for t in (w, b))
    y = ops.layer_norm(x, w, b, eps, act_bits)
    names = [(n, t) for n, t in (("dx", x), ("dw", w), ("db", b)) if t is not None]
    out = {"y": y}
    out.update(zip([n for n, _ in names], torch.autograd.grad(y, [t for _, t in names], g)))
    return out


LN_SHAPES = [(1, 1), (5, 2), (3, 7), (64, 8), (130, 16), (7, 31), (1000, 32), (9, 33), (259, 64), (31, 77), (66, 128), (17, 255), (40, 256), (5, 257),
             (12, 512), (6, 777), (33, 1000), (4, 1024), (3, 2048), (2, 2056), (5, 4096), (3, 4097), (2, 8200), (2, 20000), (4099, 24), (1, 4104)]


@pytest.mark.parametrize("act_bits", [0, 8])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,C", LN_SHAPES)
def test_layer_norm(rows, C, dtype, act_bits):
    g = gen(rows * 31 + C)
    x = randn(g, rows, C, dtype=DT[dtype], scale=1.5, shift=0.4)
    w, b, go = randn(g, C, scale=0.3, shift=1.0), randn(g, C), randn(g, rows, C, dtype=DT[dtype])
    check(run_layer_norm(x, w, b, 1e-5, go, act_bits), ref.layer_norm(x, w, b, 1e-5, go, act_bits), "layer_norm")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["offset", "constant", "tiny", "eps", "huge"])
def test_layer_norm_values(kind, dtype):
    """a mean far above the deviations, rows without deviation, values whose variance is below eps, a large eps, squares near the type's end"""
    g = gen(5)
    dt = DT[dtype]
    x = {"offset": randn(g, 20, 96, dtype=dt, scale=1.0, shift=200.0), "constant": torch.full((20, 96), 3.0, device="cuda", dtype=dt),
         "tiny": randn(g, 20, 96, dtype=dt, scale=1e-4), "eps": randn(g, 20, 96, dtype=dt), "huge": randn(g, 20, 96, dtype=dt, scale=1e4)}[kind]
    w, b, go = randn(g, 96), randn(g, 96), randn(g, 20, 96, dtype=dt)
    eps = 0.5 if kind == "eps" else 1e-5
    for act_bits in (0, 8):
        check(run_layer_norm(x, w, b, eps, go, act_bits), ref.layer_norm(x, w, b, eps, go, act_bits), kind)


@pytest.mark.parametrize("w,b", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_parameters(w, b):
    g = gen(6)
    x, go = randn(g, 70, 48), randn(g, 70, 48)
    w, b = randn(g, 48) if w else None, randn(g, 48) if b else None
    check(run_layer_norm(x, w, b, 1e-5, go), ref.layer_norm(x, w, b, 1e-5, go), "layer_norm")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_layer_norm_layouts(dtype):
    """cut-out columns, every other row, an odd start, a transposed axis, leading axes, an expanded gradient, parameters in the input's type"""
    from movedepth_amd import ops

    g, dt = gen(7), DT[dtype]
    base = randn(g, 40, 200, dtype=dt)
    w, b = randn(g, 64, dtype=dt), randn(g, 64, dtype=dt)
    views = [base[:, 8:72], base[::2, 3:67], base[:, 1:65], base.t()[:64].t(), base.view(-1)[5:5 + 64 * 100].view(100, 64), base.view(20, 2, 200)[:, :, :64],
             base[:, :1].expand(40, 64)]
    for x in views:
        go = randn(g, *x.shape, dtype=dt)
        for act_bits in (0, 8):
            got = run_layer_norm(x, w, b, 1e-5, go, act_bits)
            want = ref.layer_norm(x.reshape(-1, 64), w, b, 1e-5, go.reshape(-1, 64), act_bits)
            assert got["y"].shape == x.shape and got["dw"].dtype == dt
            for name in ("dw", "db"):
                want[name] = (want[name][0], want[name][1] + ref.u_of(dt) * want[name][0].abs())
            check({n: t.reshape(-1, 64) if n in ("y", "dx") else t for n, t in got.items()}, want, "view")
    x = randn(g, 6, 64, dtype=dt).requires_grad_()
    wp = randn(g, 64).requires_grad_()
    gx, gw = torch.autograd.grad(ops.layer_norm(x, wp).sum(), (x, wp))     # the gradient of sum() is one value, expanded
    want = ref.layer_norm(x, wp, None, 1e-5, torch.ones(6, 64))
    check({"dx": gx, "dw": gw}, want, "expanded gradient")


def test_layer_norm_partial_gradients_and_empty():
    from movedepth_amd import ops

    g = gen(8)
    x, w, b, go = randn(g, 50, 40), randn(g, 40), randn(g, 40), randn(g, 50, 40)
    want = ref.layer_norm(x, w, b, 1e-5, go)
    for need in ("x", "w", "b"):
        ts = {n: t.clone().requires_grad_(n == need) for n, t in (("x", x), ("w", w), ("b", b))}
        y = ops.layer_norm(ts["x"], ts["w"], ts["b"])
        check({"d" + need: torch.autograd.grad(y, ts[need], go)[0]}, want, "only " + need)
    with torch.no_grad():
        check({"y": ops.layer_norm(x, w, b)}, want, "no_grad")
    e = torch.zeros(0, 40, device="cuda", requires_grad=True)
    we = w.clone().requires_grad_()
    y = ops.layer_norm(e, we, b)
    gx, gw = torch.autograd.grad(y.sum(), (e, we))
    assert y.shape == (0, 40) and gx.shape == (0, 40) and not bool(gw.any())


def test_layer_norm_refusals():
    from movedepth_amd import ops

    x = torch.zeros(4, 8, device="cuda")
    for bad in (lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x, torch.ones(7, device="cuda")), lambda: ops.layer_norm(x, torch.ones(8)),
                lambda: ops.layer_norm(x, act_bits=4), lambda: ops.layer_norm(x, eps=-1.0), lambda: ops.layer_norm(x[:, :0]),
                lambda: ops.layer_norm(x, eps=float("nan")), lambda: ops.layer_norm(x.long()), lambda: ops.layer_norm(torch.zeros((), device="cuda"))):
        with pytest.raises(RuntimeError):
            bad()
    y = ops.layer_norm(x.requires_grad_())
    (gx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):                       # no second derivative
        gx.sum().backward()


# --------------------------------------------------------------------------- cross attention
def run_attention(q, k, v, mask, scale, g):
    from movedepth_amd import ops

    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    o = ops.cross_attention(q, k, v, mask, scale)
    out = {"o": o}
    out.update(zip(("dq", "dk", "dv"), torch.autograd.grad(o, (q, k, v), g)))
    with torch.no_grad():                                   # the inference call gives the same values
        assert torch.equal(ops.cross_attention(q, k, v, mask, scale), o)
    return out


def make_mask(kind, B, Nk, g):
    if kind == "none":
        return None
    m = torch.rand(B, Nk, generator=g) < 0.6
    if kind == "tail":
        m = torch.arange(Nk)[None, :] < torch.linspace(Nk, 1, B).long()[:, None]
    if kind == "empty":
        m[0] = False
    if kind == "single":
        m[:] = False
        m[torch.arange(B), torch.randint(0, Nk, (B,), generator=g)] = True
    if kind == "blocks":                                    # whole tiles without a key, at either end
        m[:] = False
        m[:, Nk // 3:Nk // 3 + 3] = True
    return m.cuda()


def attention_case(B, Nq, Nk, Hq, Hk, d, dtype, kind, seed=0, scale=None, qscale=1.5):
    g = gen(seed + 7 * Nq + 13 * Nk + d)
    dt = DT[dtype]
    q, go = randn(g, B, Nq, Hq, d, dtype=dt, scale=qscale), randn(g, B, Nq, Hq, d, dtype=dt)
    k, v = randn(g, B, Nk, Hk, d, dtype=dt), randn(g, B, Nk, Hk, d, dtype=dt, shift=0.2)
    mask = make_mask(kind, B, Nk, g)
    s = d ** -0.5 if scale is None else scale
    check(run_attention(q, k, v, mask, s, go), ref.cross_attention(q, k, v, mask, s, go), "B%d Nq%d Nk%d H%d/%d d%d %s %s" % (B, Nq, Nk, Hq, Hk, d, dtype, kind))


XA_SHAPES = [(1, 1, 1, 1, 1, 1), (2, 1, 37, 4, 2, 16), (2, 3, 5, 2, 2, 8), (1, 31, 33, 1, 1, 32), (2, 32, 32, 2, 1, 64), (1, 64, 65, 3, 3, 24), (2, 70, 129, 2, 2, 40),
             (1, 130, 63, 4, 1, 80), (1, 129, 257, 2, 2, 96), (3, 33, 100, 2, 1, 128), (1, 200, 7, 1, 1, 17), (1, 5, 300, 6, 2, 127), (2, 257, 128, 1, 1, 48), (1, 2, 1500, 8, 2, 64),
             (1, 1, 4100, 2, 2, 128), (1, 500, 260, 1, 1, 16), (1, 9, 700, 5, 5, 33), (4, 1, 64, 16, 1, 32), (1, 16, 2049, 1, 1, 112)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,d", XA_SHAPES)
def test_cross_attention(B, Nq, Nk, Hq, Hk, d, dtype):
    attention_case(B, Nq, Nk, Hq, Hk, d, dtype, "none")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("kind", ["random", "tail", "empty", "single", "blocks"])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,d", [(3, 40, 200, 2, 1, 32), (2, 1, 333, 4, 2, 64), (2, 150, 70, 2, 2, 16), (2, 9, 130, 2, 1, 72)])
def test_cross_attention_masks(B, Nq, Nk, Hq, Hk, d, kind, dtype):
    attention_case(B, Nq, Nk, Hq, Hk, d, dtype, kind)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("qscale,scale", [(30.0, None), (1.0, 0.0), (1.0, -0.3), (0.01, None)])
def test_cross_attention_sharp_and_flat(qscale, scale, dtype):
    """weights that are all but one-hot, equal weights, a negative scale"""
    attention_case(1, 66, 140, 2, 2, 32, dtype, "none", scale=scale, qscale=qscale)
    attention_case(2, 2, 300, 2, 1, 64, dtype, "random", scale=scale, qscale=qscale)


@pytest.mark.parametrize("Nq", [1, 6, 50])
@pytest.mark.parametrize("dtype", DT)
def test_cross_attention_rising_scores(Nq, dtype):
    """scores that grow along the keys: the running maximum moves in every tile, by little and by much"""
    g, dt = gen(11), DT[dtype]
    q = torch.ones(1, Nq, 1, 16, dtype=dt).cuda()
    for step in (0.01, 1.0, 8.0):
        k = (torch.arange(300).float()[None, :, None, None] * step / 16).expand(1, 300, 1, 16).to(dt).cuda()
        v, go = randn(g, 1, 300, 1, 16, dtype=dt), randn(g, 1, Nq, 1, 16, dtype=dt)
        check(run_attention(q, k, v, None, 1.0, go), ref.cross_attention(q, k, v, None, 1.0, go), "rising %g" % step)


@pytest.mark.parametrize("Nq", [1, 40])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf"), None])
def test_cross_attention_garbage_in_masked_rows(value, dtype, Nq):
    g, dt = gen(12), DT[dtype]
    q, go = randn(g, 2, Nq, 4, 32, dtype=dt), randn(g, 2, Nq, 4, 32, dtype=dt)
    k, v = randn(g, 2, 90, 2, 32, dtype=dt), randn(g, 2, 90, 2, 32, dtype=dt)
    mask = make_mask("empty", 2, 90, g)
    want = ref.cross_attention(q, k, v, mask, 0.2, go)
    fill = torch.finfo(dt).min if value is None else value
    k[~mask], v[~mask] = fill, fill
    got = run_attention(q, k, v, mask, 0.2, go)
    check(got, want, "garbage")
    assert not bool(got["o"][0].any()) and not bool(got["dq"][0].any()) and not bool(got["dk"][~mask].any()) and not bool(got["dv"][~mask].any())


@pytest.mark.parametrize("Nq", [1, 45])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cross_attention_layouts(dtype, Nq):
    """views of a joint projection, heads before tokens, an odd start, a cut-out head, an axis that is not contiguous, one state for every sequence, a
    strided mask, an expanded gradient"""
    g, dt = gen(13), DT[dtype]
    B, Nk, H, d = 2, 77, 2, 24
    kv = randn(g, B, Nk, 2, H, d, dtype=dt)
    q0 = randn(g, B, H, Nq, d, dtype=dt)
    flat = randn(g, B * Nq * H * d + 1, dtype=dt)
    wide = randn(g, B, Nk, H, d + 5, dtype=dt)
    one = randn(g, 1, Nk, H, d, dtype=dt)
    per = randn(g, B, d, H, Nk, dtype=dt).permute(0, 3, 2, 1)
    big = torch.rand(B, 2 * Nk, generator=g).cuda() < 0.7
    go = randn(g, B, Nq, H, d, dtype=dt)
    qs = [q0.transpose(1, 2), flat[1:].view(B, Nq, H, d)]
    kvs = [(kv[:, :, 0], kv[:, :, 1]), (wide[..., :d], wide[..., 3:3 + d]), (one.expand(B, Nk, H, d), kv[:, :, 1]), (per, per), (kv[:, :, 0].flip(1), one.expand(B, Nk, H, d)),
           (kv[:, :, 0, :1].expand(B, Nk, H, d), kv[:, :, 1])]
    for q in qs:
        for k, v in kvs:
            for mask in (None, big[:, ::2], big[:1, :Nk].expand(B, Nk)):
                check(run_attention(q, k, v, mask, 0.25, go), ref.cross_attention(q, k, v, mask, 0.25, go), "layout")
    from movedepth_amd import ops
    q, k, v = (t.detach().clone().requires_grad_() for t in (qs[0], *kvs[0]))
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(ops.cross_attention(q, k, v).sum(), (q, k, v))))
    check(got, ref.cross_attention(q, k, v, None, d ** -0.5, torch.ones(B, Nq, H, d)), "expanded gradient")


def test_cross_attention_broadcast_state_gradient():
    """one encoder state for every sequence: autograd's expand sums the gradients of the shared rows"""
    from movedepth_amd import ops

    g = gen(14)
    q, go = randn(g, 3, 20, 4, 16), randn(g, 3, 20, 4, 16)
    k1, v1 = randn(g, 1, 50, 2, 16).requires_grad_(), randn(g, 1, 50, 2, 16).requires_grad_()
    o = ops.cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1))
    dk, dv = torch.autograd.grad(o, (k1, v1), go)
    want = ref.cross_attention(q, k1.expand(3, -1, -1, -1), v1.expand(3, -1, -1, -1), None, 0.25, go)
    for name, t in (("dk", dk), ("dv", dv)):
        val, tol = want[name]
        ref.within(t, val.sum(0, keepdim=True), tol.sum(0, keepdim=True) + 3 * 2.0 ** -24 * val.abs().sum(0, keepdim=True), name)


def test_cross_attention_empty_sizes():
    from movedepth_amd import ops

    for B, Nq, Nk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k, v = (torch.ones(B, n, 2, 16, device="cuda", requires_grad=True) for n in (Nq, Nk, Nk))
        o = ops.cross_attention(q, k, v)
        assert o.shape == (B, Nq, 2, 16) and not bool(o.any())
        for t, gr in zip((q, k, v), torch.autograd.grad(o.sum(), (q, k, v))):
            assert gr.shape == t.shape and not bool(gr.any())


def test_cross_attention_partial_gradients():
    from movedepth_amd import ops

    g = gen(15)
    q, k, v, go = randn(g, 1, 40, 2, 32), randn(g, 1, 60, 2, 32), randn(g, 1, 60, 2, 32), randn(g, 1, 40, 2, 32)
    want = ref.cross_attention(q, k, v, None, 32 ** -0.5, go)
    for need in ("q", "k", "v"):
        ts = {n: t.clone().requires_grad_(n == need) for n, t in (("q", q), ("k", k), ("v", v))}
        check({"d" + need: torch.autograd.grad(ops.cross_attention(**ts), ts[need], go)[0]}, want, "only " + need)


def test_cross_attention_refusals():
    from movedepth_amd import ops

    def t(*s, dtype=torch.float32):
        return torch.zeros(*s, device="cuda", dtype=dtype)

    q, k = t(1, 3, 4, 16), t(1, 5, 2, 16)
    bad = [(q, k, t(1, 6, 2, 16)), (q, t(1, 5, 3, 16), t(1, 5, 3, 16)), (q, t(2, 5, 2, 16), t(2, 5, 2, 16)), (q, t(1, 5, 2, 8), t(1, 5, 2, 8)), (t(1, 3, 2, 129), t(1, 5, 2, 129), t(1, 5, 2, 129)),
           (q.double(), k.double(), k.double()), (q, k.bfloat16(), k), (q[0], k[0], k[0]), (q, k, k.cpu()), (t(1, 3, 2, 0), t(1, 5, 2, 0), t(1, 5, 2, 0)), (q, t(1, 5, 0, 16), t(1, 5, 0, 16))]
    for a in bad:
        with pytest.raises(RuntimeError):
            ops.cross_attention(*a)
    for m in (t(1, 5), t(1, 4, dtype=torch.bool), t(2, 5, dtype=torch.bool), torch.zeros(1, 5, dtype=torch.bool), t(5, dtype=torch.bool)):
        with pytest.raises(RuntimeError):
            ops.cross_attention(q, k, k, key_mask=m)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,d", [(1, 12, 9000, 1, 1, 32), (2, 5, 5000, 4, 2, 64), (1, 3000, 40, 2, 1, 16), (3, 33, 1200, 1, 1, 128)])
def test_cross_attention_long_axes(B, Nq, Nk, Hq, Hk, d, dtype):
    """few rows against many: the work of a block of rows is spread over many workgroups and joined"""
    attention_case(B, Nq, Nk, Hq, Hk, d, dtype, "none")
    attention_case(B, Nq, Nk, Hq, Hk, d, dtype, "tail")


@pytest.mark.parametrize("size", [1e-4, 1.0, 300.0])
def test_cross_attention_float16_gradient_sizes(size):
    """gradients far below and above 1: dS of a long row would fall below float16's range, or above it.  Relative to the largest: the scaled dS keeps 2^-25 of
    2^15 / (2 |g| |v|), so what is lost is below 2^-40 of |g| |v| per key, under the bound's own terms; the results themselves must fit the type"""
    g = gen(40)
    q, k, v = randn(g, 1, 70, 2, 32, dtype=torch.float16), randn(g, 1, 400, 2, 32, dtype=torch.float16), randn(g, 1, 400, 2, 32, dtype=torch.float16)
    go = randn(g, 1, 70, 2, 32, dtype=torch.float16, scale=size)
    got = run_attention(q, k, v, None, 0.2, go)
    check(got, ref.cross_attention(q, k, v, None, 0.2, go), "gradient of size %g" % size)
    if size < 1:                # 1024 times the gradient gives 1024 times the gradients, but for the small ones' own last step
        big = run_attention(q, k, v, None, 0.2, go * 1024)
        for name in ("dq", "dk", "dv"):
            a, b = got[name].double() * 1024, big[name].double()
            assert bool(((a - b).abs() <= 1024 * ref.tiny_of(torch.float16) + 2 * ref.u_of(torch.float16) * b.abs()).all()), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_cross_attention_where_the_norms_bound_the_scores_and_where_not(dtype):
    """rows and keys of very different sizes in one call: some blocks of rows run without a running maximum, some with, and parts of both are joined"""
    g, dt = gen(41), DT[dtype]
    q = randn(g, 1, 400, 1, 32) * torch.where(torch.arange(400) < 200, 0.3, 12.0)[None, :, None, None].cuda()
    k = randn(g, 1, 2000, 1, 32) * torch.where(torch.arange(2000) < 900, 0.5, 4.0)[None, :, None, None].cuda()
    v, go = randn(g, 1, 2000, 1, 32, dtype=dt), randn(g, 1, 400, 1, 32, dtype=dt)
    q, k = q.to(dt), k.to(dt)
    check(run_attention(q, k, v, None, 0.4, go), ref.cross_attention(q, k, v, None, 0.4, go), "mixed norms")
    k = -k.abs()                                            # every score far below 0
    q = q.abs()
    check(run_attention(q, k, v, None, 0.4, go), ref.cross_attention(q, k, v, None, 0.4, go), "low scores")


@pytest.mark.parametrize("Nq", [1, 40])
def test_cross_attention_offsets_beyond_32_bits(Nq):
    """rows of a cache whose last offset passes 2^32 elements"""
    from movedepth_amd import ops

    g = gen(16)
    step = (1 << 32) // 63 + 64
    step -= step % 8
    store = torch.empty(64 * step + 64, device="cuda", dtype=torch.bfloat16)
    k = store.as_strided((1, 64, 1, 32), (0, step, 32, 1))
    v = store.as_strided((1, 64, 1, 32), (0, step, 32, 1), 32)
    k.copy_(randn(g, 1, 64, 1, 32, dtype=torch.bfloat16))
    v.copy_(randn(g, 1, 64, 1, 32, dtype=torch.bfloat16))
    q, go = randn(g, 1, Nq, 1, 32, dtype=torch.bfloat16), randn(g, 1, Nq, 1, 32, dtype=torch.bfloat16)
    check(run_attention(q, k, v, None, 0.2, go), ref.cross_attention(q, k.clone(), v.clone(), None, 0.2, go), "long cache")


# --------------------------------------------------------------------------- differences, repetition, streams, graphs
@pytest.mark.parametrize("op", ["layer_norm", "cross_attention"])
def test_gradients_against_differences(op):
    """the derivative along a direction against central differences of the 32-bit forward pass: Richardson's remainder from two steps, and the
    forward pass's own bound divided by the step"""
    from movedepth_amd import ops

    g = gen(17)
    if op == "layer_norm":
        ins = [randn(g, 10, 48), randn(g, 48), randn(g, 48)]
        f, bound = (lambda *a: ops.layer_norm(*a)), (lambda *a: ref.layer_norm(*a, 1e-5)["y"][1])
    else:
        ins = [randn(g, 1, 40, 2, 16), randn(g, 1, 50, 2, 16), randn(g, 1, 50, 2, 16)]
        f, bound = (lambda *a: ops.cross_attention(*a)), (lambda *a: ref.cross_attention(*a, None, 0.25)["o"][1])
    go = torch.randn(f(*ins).shape, generator=g)
    for i in range(3):
        leaf = [t.clone().requires_grad_(j == i) for j, t in enumerate(ins)]
        (gr,) = torch.autograd.grad(f(*leaf), leaf[i], go.cuda())
        u = torch.randn(ins[i].shape, generator=g).cuda()

        def at(h):
            # the step that 32 bits really make
            p, m = ins[i] + h * u, ins[i] - h * u
            fp, fm = (f(*[t if j == i else s for j, s in enumerate(ins)]).double().cpu() for t in (p, m))
            return float(((fp - fm) * go.double()).sum()), (p.double() - m.double()).cpu()

        h = 2.0 ** -6
        (l1, s1), (l2, s2) = at(h), at(2 * h)
        d1, d2 = l1, l2 / 2
        want = float((gr.double().cpu() * s1).sum())
        noise = 2 * float((go.double().abs() * bound(*ins)).sum())
        assert abs(want - d1) <= abs(d2 - d1) + 3 * noise + 1e-4 * abs(d1), "%s input %d: %.6g, by differences %.6g" % (op, i, want, d1)


def operators(g, dt=torch.bfloat16, d=32):
    """closures that make every kernel of the operators run once on fixed inputs -> (inputs, function of them)"""
    from movedepth_amd import ops

    x, w, b, gx = randn(g, 300, 96, dtype=dt), randn(g, 96), randn(g, 96), randn(g, 300, 96, dtype=dt)
    q, k, v, go = randn(g, 2, 140, 4, d, dtype=dt), randn(g, 2, 210, 2, d, dtype=dt), randn(g, 2, 210, 2, d, dtype=dt), randn(g, 2, 140, 4, d, dtype=dt)
    q1 = randn(g, 2, 1, 4, d, dtype=dt)
    mask = make_mask("random", 2, 210, g)

    def f(x, w, b, gx, q, k, v, go, q1):
        out = list(run_layer_norm(x, w, b, 1e-5, gx, 8).values()) + list(run_layer_norm(x, w, b, 1e-5, gx).values())
        out.append(ops.act8_unpack(ops.act8_pack(x)))
        qq, kk, vv = (t.detach().requires_grad_() for t in (q, k, v))
        o = ops.cross_attention(qq, kk, vv, mask)
        out += [o.detach(), *torch.autograd.grad(o, (qq, kk, vv), go)]
        with torch.no_grad():
            out += [ops.cross_attention(q1, k, v, mask), ops.cross_attention(q1, k, v)]
        return [t.detach() for t in out]

    return [x, w, b, gx, q, k, v, go, q1], f


@pytest.mark.parametrize("dtype", DT)
def test_same_bits_every_time(dtype):
    ins, f = operators(gen(18), DT[dtype])
    first = [t.clone() for t in f(*ins)]
    junk = torch.full((1 << 22,), float("nan"), device="cuda")       # what the next workspaces are cut from
    del junk
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, f(*ins)))


def test_another_stream():
    ins, f = operators(gen(19))
    want = [t.clone() for t in f(*ins)]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = f(*ins)
    b = f(*ins)                                               # at the same time on the current stream
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) and torch.equal(x, z) for x, y, z in zip(want, a, b))


@pytest.mark.parametrize("dtype,d", [("bf16", 32), ("f32", 128), ("f16", 64)])
def test_captured_graphs(dtype, d):
    """two graphs of one memory pool, replayed in turn with new inputs and eager work between"""
    ins, f = operators(gen(20), DT[dtype], d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        f(*ins)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs, outs, pool = [], [], None
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(f(*ins))
        pool = g.pool()
        graphs.append(g)
    for i in range(4):
        new, _ = operators(gen(30 + i), DT[dtype], d)
        for t, n in zip(ins, new):
            t.copy_(n)
        want = [t.clone() for t in f(*ins)]
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, out)), "replay %d" % i


# --------------------------------------------------------------------------- the operators together
def match_attention_64(m, x, others, go):
    """MatchAttention in 64 bits on the CPU, from the operators' definitions; gradients by autograd"""
    P = {n: p.detach().double().cpu().requires_grad_() for n, p in m.named_parameters()}
    x, others = x.detach().double().cpu().requires_grad_(), [o.detach().double().cpu().requires_grad_() for o in others]
    B, C, h, w = x.shape
    tok = lambda t: t.permute(0, 2, 3, 1).flatten(1, 2)  # noqa: E731
    ln = lambda t: torch.nn.functional.layer_norm(t, (C,), P["norm.weight"], P["norm.bias"], m.norm.eps)  # noqa: E731
    q = (ln(tok(x)) @ P["q.weight"].t()).view(B, h * w, m.heads, -1).transpose(1, 2)
    kv = (ln(torch.cat([tok(o) for o in others], 1)) @ P["kv.weight"].t()).view(B, -1, 2, m.heads, C // m.heads).permute(2, 0, 3, 1, 4)
    a = torch.softmax(q @ kv[0].transpose(2, 3) * (C // m.heads) ** -0.5, 3) @ kv[1]
    y = x + (a.transpose(1, 2).reshape(B, h * w, C) @ P["out.weight"].t()).view(B, h, w, C).permute(0, 3, 1, 2)
    grads = torch.autograd.grad(y, [x] + others + list(P.values()), go.double().cpu())
    return [y] + list(grads)


@pytest.mark.parametrize("act_bits", [0, 8])
@pytest.mark.parametrize("frames", [1, 2])
def test_match_attention(frames, act_bits):
    """the block that the trainer puts ahead of the plane sweep: forward and every gradient.  32 bits through four products, two norms and a softmax: 1e-4 norm-wise,
    as the other operators of the step; with the norms' inputs in 8 bits each is off by at most 2^-7 of its group's largest, whose square is
    at least the mean square of the group, so by less than 2^-7 sqrt(32) of the row norm-wise at the very worst, half a step on average: 2 %"""
    from movedepth_amd import networks

    torch.manual_seed(0)
    m = networks.MatchAttention(32, 2, act_bits).cuda()
    torch.nn.init.normal_(m.out.weight, std=0.2)
    g = gen(21)
    x = randn(g, 2, 32, 9, 14).contiguous(memory_format=torch.channels_last).requires_grad_()
    others = [randn(g, 2, 32, 9, 14).contiguous(memory_format=torch.channels_last).requires_grad_() for _ in range(frames)]
    go = randn(g, 2, 32, 9, 14)
    y = m(x, others)
    assert y.is_contiguous(memory_format=torch.channels_last)
    got = [y] + list(torch.autograd.grad(y, [x] + others + list(m.parameters()), go))
    want = match_attention_64(m, x, others, go)
    for i, (a, b) in enumerate(zip(got, want)):
        err = float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())
        assert err <= (1e-4 if i == 0 or not act_bits else 2e-2), "result %d is off by %.3g" % (i, err)


def step(extra, dtype=None, models=None):
    """one training step of the real trainer -> (losses, gradients by name, trainer)"""
    from movedepth_amd.options import MovedepthOptions
    from movedepth_amd.synthetic import make_inputs
    from movedepth_amd.trainer import Trainer

    opt = MovedepthOptions().parse(["--height", "64", "--width", "128", "--num_depth_bins", "16", "--batch_size", "2", "--convex_up", "--weights_init", "scratch",
                                    "--miopen_find", "0", "--automask_noise", "host"] + extra)
    torch.manual_seed(3)
    t = Trainer(opt)
    if models is not None:
        for n, m in models.items():
            t.models[n].load_state_dict(m)
    t.set_train()
    torch.manual_seed(4)
    np.random.seed(4)
    random.seed(4)
    with torch.autocast("cuda", dtype=dtype) if dtype is not None else contextlib.nullcontext():
        outputs, losses = t.process_batch(make_inputs(2, 64, 128, opt.frame_ids, seed=5, device=t.device), is_train=True)
    losses["loss"].backward()
    return losses, {"%s.%s" % (n, k): p.grad for n, m in t.models.items() for k, p in m.named_parameters()}, t


def test_trainer_with_match_attention_and_8_bit_activations(tmp_path):
    """the untrained block hands the features through: the step's loss is the plain step's; its gradients run; checkpoints carry it; 2-byte features work"""
    _, _, plain = step([])
    state = {n: m.state_dict() for n, m in plain.models.items()}
    base, g0, _ = step([], models=state)
    losses, g1, t = step(["--match_attention", "2"], models=state)
    assert "match_attn" not in plain.models and "match_attn" in t.models
    assert abs(float(losses["loss"].detach()) - float(base["loss"].detach())) <= 1e-4 * abs(float(base["loss"].detach()))
    assert g1["match_attn.out.weight"] is not None and bool(g1["match_attn.out.weight"].any()) and bool(torch.isfinite(g1["match_attn.out.weight"]).all())
    trained = {**state, "match_attn": t.models["match_attn"].state_dict()}
    torch.nn.init.normal_(t.models["match_attn"].out.weight, std=0.2)
    trained = {**state, "match_attn": t.models["match_attn"].state_dict()}
    full, gf, _ = step(["--match_attention", "2"], models=trained)
    kept, g8, t8 = step(["--match_attention", "2", "--act_bits", "8"], models=trained)
    assert abs(float(full["loss"].detach()) - float(kept["loss"].detach())) <= 1e-4 * abs(float(full["loss"].detach()))   # the forward pass does not change
    for n in gf:
        if n.startswith("match_attn"):
            assert bool(gf[n].any()) and bool(torch.isfinite(gf[n]).all()) and bool(torch.isfinite(g8[n]).all()), n
    half, gh, _ = step(["--match_attention", "2", "--act_bits", "8"], dtype=torch.bfloat16, models=trained)
    assert bool(torch.isfinite(half["loss"])) and all(bool(torch.isfinite(v).all()) for n, v in gh.items() if n.startswith("match_attn"))
    t8.opt.log_dir, t8.log_path = str(tmp_path), str(tmp_path / "m")
    t8.save_model()
    t8.opt.load_weights_folder = str(tmp_path / "m" / "models" / "weights_0")
    before = t8.models["match_attn"].out.weight.detach().clone()
    with torch.no_grad():
        t8.models["match_attn"].out.weight.zero_()
    t8.load_model()
    assert torch.equal(t8.models["match_attn"].out.weight, before)


def test_evaluation_with_match_attention():
    from movedepth_amd.evaluate_depth import predict_depth
    from movedepth_amd.synthetic import make_inputs

    _, _, t = step(["--match_attention", "2"])
    t.set_eval()
    data = make_inputs(2, 64, 128, t.opt.frame_ids, seed=6)
    a = predict_depth(t.models, data, t.opt, t.vol_layout)["depth_mvs"]
    torch.nn.init.normal_(t.models["match_attn"].out.weight, std=0.2)
    b = predict_depth(t.models, data, t.opt, t.vol_layout)["depth_mvs"]
    del t.models["match_attn"]
    c = predict_depth(t.models, data, t.opt, t.vol_layout)["depth_mvs"]
    assert torch.allclose(a, c, rtol=1e-4) and not torch.allclose(b, c, rtol=1e-4) and bool(torch.isfinite(b).all())


def test_cross_attention_many_sequences():
    """more masked sequences than a wave has lanes, of every number of valid keys, some without any"""
    g = gen(50)
    q, go = randn(g, 150, 10, 1, 16), randn(g, 150, 10, 1, 16)
    k, v = randn(g, 150, 70, 1, 16), randn(g, 150, 70, 1, 16)
    mask = (torch.arange(70)[None, :] < torch.randint(0, 71, (150,), generator=g)[:, None]).cuda()
    mask[60:70] = False
    mask[0] = False
    check(run_attention(q, k, v, mask, 0.25, go), ref.cross_attention(q, k, v, mask, 0.25, go), "many sequences")


def test_more_than_one_launch_holds():
    """a launch takes 2^32 elements of act8_pack and 2^20 long rows of layer_norm: what lies behind them is the next launch's.  Elements and rows are
    independent of each other, so those on both sides of the seam have the bits that a call of theirs alone gives."""
    from movedepth_amd import ops

    g = gen(51)
    n, edge = (1 << 32) + 100, 4096
    x = torch.ones(n, device="cuda", dtype=torch.bfloat16)
    around = torch.cat([randn(g, edge).bfloat16(), randn(g, 100).bfloat16()])
    x[n - edge - 100:] = around
    p, few = ops.act8_pack(x), ops.act8_pack(around)
    back = ops.act8_unpack(p)
    assert torch.equal(p.codes[n - edge - 100:], few.codes) and torch.equal(p.scales[-few.scales.numel():], few.scales)
    assert torch.equal(back[n - edge - 100:], ops.act8_unpack(few)) and bool((back[:n - edge - 100] == 1).all())
    del x, p, back
    rows, C = (1 << 20) + 3, 8193
    at = torch.tensor([0, 1, (1 << 20) - 1, 1 << 20, (1 << 20) + 2], device="cuda")
    few, go = randn(g, 5, C).bfloat16().requires_grad_(), randn(g, 5, C).bfloat16()
    x, gy = torch.ones(rows, C, device="cuda", dtype=torch.bfloat16), torch.zeros(rows, C, device="cuda", dtype=torch.bfloat16)
    x[at], gy[at] = few.detach(), go
    w = randn(g, C)
    for act_bits in (0, 8):
        y = ops.layer_norm(x.requires_grad_(), w, None, 1e-5, act_bits)
        y1 = ops.layer_norm(few, w, None, 1e-5, act_bits)
        dx, = torch.autograd.grad(y, x, gy)
        dx1, = torch.autograd.grad(y1, few, go)
        assert torch.equal(y.detach()[at], y1) and torch.equal(dx[at], dx1)
        assert not bool(y.detach()[2:(1 << 20) - 1].any()) and not bool(dx[2:(1 << 20) - 1].any())      # constant rows, no gradient
        del y, dx
