"""The token operators' refusals at the C boundary and in Python (before any launch: no GPU), their CPU path in the module, and the definitions the GPU
tests hold them to."""
import ctypes

import pytest
import torch

import token_ref as ref


def desc(**kw):
    from movedepth_amd import _lib

    a = _lib.AttnDesc()
    a.dtype, a.B, a.Nq, a.Nk, a.Hq, a.Hk, a.d, a.scale = 0, 1, 2, 3, 2, 1, 16, 0.25
    for n in ("q", "k", "v", "o", "lse", "g", "dq", "dk", "dv"):
        setattr(a, n, 4096)
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def refused(rc, *words):
    from movedepth_amd import _lib

    msg = _lib.load().md_last_error().decode()
    assert rc == -1, rc
    for w in words:
        assert w in msg, msg


def test_layer_norm_refuses():
    from movedepth_amd import _lib

    lib = _lib.load()
    fwd = lambda **k: lib.md_layer_norm_fwd(*{**dict(x=64, dtype=0, rows=2, C=8, ldx=8, w=None, b=None, eps=1e-5, y=64, stat=None, codes=None, scales=None, s=None), **k}.values())  # noqa: E731
    refused(fwd(x=None), "md_layer_norm_fwd", "null")
    refused(fwd(y=None), "null")
    refused(fwd(dtype=3), "dtype")
    refused(fwd(C=0), "columns")
    refused(fwd(C=(1 << 20) + 1, ldx=1 << 21), "columns")
    refused(fwd(rows=-1), "rows")
    refused(fwd(rows=1 << 31), "rows")
    refused(fwd(ldx=7), "stride")
    refused(fwd(eps=-1.0), "eps")
    refused(fwd(eps=float("nan")), "eps")
    refused(fwd(codes=64), "come together")
    assert fwd(rows=0) == 0
    bwd = lambda **k: lib.md_layer_norm_bwd(*{**dict(g=64, ldg=8, x=64, ldx=8, codes=None, scales=None, dtype=0, stat=64, w=None, rows=2, C=8, dx=64, dw=64, db=64, ws=64, n=1 << 20, s=None), **k}.values())  # noqa: E731
    refused(bwd(g=None), "md_layer_norm_bwd", "null")
    refused(bwd(x=None), "null")
    refused(bwd(stat=None), "null")
    refused(bwd(dtype=-1), "dtype")
    refused(bwd(ldg=7), "stride")
    refused(bwd(ldx=7), "stride")
    refused(bwd(n=1), "workspace")
    refused(bwd(ws=None), "workspace")
    refused(bwd(scales=64), "come together")
    assert lib.md_layer_norm_bwd_ws_bytes(0, 8) == 0 and lib.md_layer_norm_bwd_ws_bytes(5, 8) > 0


def test_act8_refuses():
    from movedepth_amd import _lib

    lib = _lib.load()
    refused(lib.md_act8_pack(None, 0, 4, 64, 64, None), "md_act8_pack", "null")
    refused(lib.md_act8_pack(64, 0, 4, None, 64, None), "null")
    refused(lib.md_act8_pack(64, 3, 4, 64, 64, None), "dtype")
    refused(lib.md_act8_pack(64, 0, -1, 64, 64, None), "negative")
    refused(lib.md_act8_pack(64, 0, (1 << 38) + 1, 64, 64, None), "elements")
    refused(lib.md_act8_unpack(64, None, 0, 4, 64, None), "md_act8_unpack", "null")
    refused(lib.md_act8_unpack(64, 64, 7, 4, 64, None), "dtype")
    refused(lib.md_act8_unpack(64, 64, 0, -4, 64, None), "negative")
    assert lib.md_act8_pack(None, 0, 0, None, None, None) == 0 and lib.md_act8_unpack(None, None, 0, 0, None, None) == 0


@pytest.mark.parametrize("entry", ["md_cross_attn_fwd", "md_cross_attn_bwd"])
def test_cross_attention_refuses(entry):
    from movedepth_amd import _lib

    f = getattr(_lib.load(), entry)
    call = lambda **k: f(ctypes.byref(desc(**k)), 4096, 1 << 40, None)  # noqa: E731
    refused(f(None, None, 0, None), entry, "null")
    refused(call(dtype=3), "dtype")
    refused(call(d=0), "head size")
    refused(call(d=129), "head size")
    refused(call(Hq=3, Hk=2), "multiple")
    refused(call(Hq=0), "multiple")
    refused(call(Hk=0), "multiple")
    refused(call(Nq=-1), "negative")
    refused(call(B=-1), "negative")
    refused(call(B=1 << 17), "65535")
    refused(call(B=60000, Hq=60000, Hk=60000, Nq=0, Nk=0), "2^31")
    refused(call(B=60000, Hq=300, Hk=300, Nq=0, Nk=0), "2^24")
    refused(call(scale=float("nan")), "scale")
    refused(call(q=None), "null")
    refused(call(k=None), "null")
    refused(call(v=None), "null")
    refused(call(o=None), "null")
    assert call(B=0) == 0
    if entry.endswith("bwd"):
        refused(call(g=None), "null")
        refused(call(lse=None), "null")
        refused(call(dk=None), "come together")
    need = _lib.load().md_cross_attn_ws_bytes(ctypes.byref(desc(Nq=300, Nk=500)), int(entry.endswith("bwd")))
    if need:
        refused(f(ctypes.byref(desc(Nq=300, Nk=500)), 4096, need - 1, None), "workspace")
        refused(f(ctypes.byref(desc(Nq=300, Nk=500)), None, need, None), "workspace")


def test_python_refuses_cpu_tensors():
    from movedepth_amd import _lib, ops

    x = torch.zeros(2, 3, 2, 16)
    for call in (lambda: ops.layer_norm(x), lambda: ops.act8_pack(x), lambda: ops.cross_attention(x, x, x)):
        with pytest.raises(_lib.MovedepthHipError, match="GPU tensor"):
            call()


def test_saved_act8_leaves_cpu_tensors_alone():
    from movedepth_amd import ops

    x = torch.randn(40, 40, requires_grad=True)
    with ops.saved_act8(min_numel=1):
        y = (x * 2) * (x + 1)
    plain = (x * 2) * (x + 1)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], torch.autograd.grad(plain.sum(), x)[0])


@pytest.mark.parametrize("shape,perm,dense", [((2, 3, 4), None, True), ((2, 3, 4), (2, 0, 1), True), ((2, 1, 4), (1, 2, 0), True), ((0, 3), None, True), ((), None, True)])
def test_dense_views(shape, perm, dense):
    from movedepth_amd import ops

    t = torch.zeros(shape)
    assert ops._is_dense(t if perm is None else t.permute(perm)) is dense
    b = torch.zeros(4, 6)
    assert not ops._is_dense(b[:, ::2]) and not ops._is_dense(b[:, :3]) and not ops._is_dense(b[:1].expand(4, 6)) and ops._is_dense(b[1:3])


def test_layer_norm_module_on_the_cpu():
    from movedepth_amd import networks

    m, t = networks.LayerNorm(24), torch.nn.LayerNorm(24)
    assert sorted(m.state_dict()) == sorted(t.state_dict())
    x = torch.randn(3, 5, 24)
    assert torch.equal(m(x), t(x))
    with pytest.raises(ValueError):
        networks.MatchAttention(32, 3)


def test_options_are_off_by_default():
    from movedepth_amd.options import MovedepthOptions
    from movedepth_amd.trainer import build_models

    opt = MovedepthOptions().parse(["--weights_init", "scratch"])
    assert opt.match_attention == 0 and opt.act_bits == 0 and "match_attn" not in build_models(opt)[0]
    opt = MovedepthOptions().parse(["--weights_init", "scratch", "--match_attention", "4", "--act_bits", "8"])
    models, _, mvs = build_models(opt)
    assert models["match_attn"].heads == 4 and models["match_attn"].norm.act_bits == 8 and mvs[-1] == "match_attn"


# the definitions themselves, where a plainer statement exists
def test_reference_layer_norm_is_torchs():
    g = torch.Generator().manual_seed(0)
    x, w, b, go = (torch.randn(s, generator=g) for s in ((6, 40), (40,), (40,), (6, 40)))
    out = ref.layer_norm(x, w, b, 1e-5, go)
    xd, wd, bd = (t.double().requires_grad_() for t in (x, w, b))
    y = torch.nn.functional.layer_norm(xd, (40,), wd, bd, 1e-5)
    for name, t in zip(("y", "dx", "dw", "db"), (y, *torch.autograd.grad(y, (xd, wd, bd), go.double()))):
        assert torch.allclose(out[name][0], t, rtol=1e-10, atol=1e-12), name


def test_reference_cross_attention_is_autograds():
    g = torch.Generator().manual_seed(1)
    q, go = torch.randn(2, 5, 4, 8, generator=g), torch.randn(2, 5, 4, 8, generator=g)
    k, v = torch.randn(2, 7, 2, 8, generator=g), torch.randn(2, 7, 2, 8, generator=g)
    mask = torch.rand(2, 7, generator=g) < 0.6
    mask[0, 0] = True
    mask[1] = False
    out = ref.cross_attention(q, k, v, mask, 0.3, go)
    qd, kd, vd = (t.double().requires_grad_() for t in (q, k, v))
    s = torch.einsum("bqhd,bkhd->bhqk", qd[:1], kd[:1].repeat_interleave(2, 2)) * 0.3
    p = torch.softmax(s.masked_fill(~mask[:1, None, None], float("-inf")), 3)
    o = torch.einsum("bhqk,bkhd->bqhd", p, vd[:1].repeat_interleave(2, 2))
    grads = torch.autograd.grad(o, (qd, kd, vd), go[:1].double())
    for name, t in zip(("o", "dq", "dk", "dv"), (o, *grads)):
        assert torch.allclose(out[name][0][:1], t[:1], rtol=1e-10, atol=1e-12), name
        assert not bool(out[name][0][1].any()), name


def test_reference_act8():
    x = torch.tensor([[127.0, 1.0, 0.5, -3.0], [127.5, 0.5, 1.5, 1.0], [255.0, 1.0, 3.0, 5.0]])
    y = ref.act8(x)
    assert y[0].tolist() == [127.0, 1.0, 0.0, -3.0] and y[1].tolist() == [128.0, 0.0, 2.0, 0.0] and y[2].tolist() == [256.0, 0.0, 4.0, 4.0]
