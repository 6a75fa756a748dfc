"""Token operators where a call can go wrong without failing: their statistics and a module's weights inside the 8-bit context, scores of minus infinity and values
that three bf16 pieces cannot hold, float16 gradients of very different sizes in one call, rows without deviation far from zero, forward-mode
tangents, and what the trainer builds from them."""
import pytest
import torch

import test_token_ops_gpu as base
import token_ref as ref

pytestmark = pytest.mark.gpu

DT, gen, randn, check = base.DT, base.gen, base.randn, base.check


def relative(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return float((got - want).norm() / want.norm())


# --------------------------------------------------------------------------- the 8-bit context
@pytest.mark.parametrize("act_bits", [0, 8])
def test_saved_act8_leaves_layer_norms_statistics(act_bits):
    """the rows' means and deviations stay in 32 bits whatever the context's limit: what is kept of x is its 8-bit value, as with act_bits=8 (rows of 64: the
    same groups of 32), and nothing else changes"""
    from movedepth_amd import ops

    g = gen(1)
    x, w, b, go = randn(g, 300, 64, shift=3.0).requires_grad_(), randn(g, 64).requires_grad_(), randn(g, 64).requires_grad_(), randn(g, 300, 64)
    with ops.saved_act8(min_numel=1):
        y = ops.layer_norm(x * 1.0, w, b, 1e-5, act_bits)
    got = dict(zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), go)), y=y)
    check(got, ref.layer_norm(x, w, b, 1e-5, go, 8), "layer_norm in the 8-bit context")


def test_saved_act8_leaves_the_statistics_of_many_rows():
    """as many rows as bring the statistics to the context's default limit"""
    from movedepth_amd import ops

    g = gen(2)
    x, go = randn(g, 1 << 19, 32, shift=3.0).requires_grad_(), randn(g, 1 << 19, 32)
    want, = torch.autograd.grad(ops.layer_norm(x, act_bits=8), x, go)
    with ops.saved_act8():
        y = ops.layer_norm(x * 1.0)
    got, = torch.autograd.grad(y, x, go)
    assert relative(got, want) <= 8 * ref.U32                # the same formula on the same 8-bit values and statistics


@pytest.mark.parametrize("B,Nq,Nk,Hq,Hk,d,limit", [(3, 21, 50, 2, 1, 16, 1), (8, 8192, 40, 16, 4, 8, 1 << 20)])
def test_saved_act8_leaves_cross_attentions_statistics(B, Nq, Nk, Hq, Hk, d, limit):
    """what is kept of q, k, v and o is their 8-bit value, the row sums stay: the gradients are the formula's on those values (in 64 bits below; the exponents' error,
    2^-24 times scores of up to ~64, and sums of up to 2^15 terms leave 1e-4 norm-wise).  A sequence without keys lies between the others: its
    rows' infinite sums must not reach a neighbour"""
    from movedepth_amd import ops

    g = gen(3)
    q, k, v = (randn(g, B, n, h, d, scale=s).requires_grad_() for n, h, s in ((Nq, Hq, 2.0), (Nk, Hk, 2.0), (Nk, Hk, 1.0)))
    go = randn(g, B, Nq, Hq, d)
    mask = (torch.rand(B, Nk, generator=g) < 0.8).cuda()
    mask[1] = False
    with ops.saved_act8(min_numel=limit):
        o = ops.cross_attention(q * 1.0, k * 1.0, v * 1.0, mask, 0.5)
    got = torch.autograd.grad(o, (q, k, v), go)

    def kept(t):
        t = t.detach()
        return (ops.act8_unpack(ops.act8_pack(t)) if t.numel() >= limit else t).double()

    G, live = Hq // Hk, mask[:, None, None, :]
    head = lambda t, r: t.transpose(1, 2).repeat_interleave(r, 1)  # noqa: E731
    s = 0.5 * head(q.detach().double(), 1) @ head(k.detach().double(), G).transpose(2, 3).contiguous()
    lse = s.masked_fill(~live, float("-inf")).logsumexp(3, keepdim=True)
    q8, k8, v8, o8, g64 = head(kept(q), 1), head(kept(k), G), head(kept(v), G), head(kept(o), 1), head(go.double(), 1)
    p = torch.where(live & torch.isfinite(lse), torch.exp(0.5 * q8 @ k8.transpose(2, 3).contiguous() - lse), 0.0)
    ds = p * (g64 @ v8.transpose(2, 3).contiguous() - (g64 * o8).sum(3, keepdim=True)) * 0.5
    shared = lambda t: t.view(B, Hk, G, Nk, d).sum(2)  # noqa: E731
    want = [ds @ k8, shared(ds.transpose(2, 3).contiguous() @ q8), shared(p.transpose(2, 3).contiguous() @ g64)]
    for name, a, b in zip(("dq", "dk", "dv"), got, want):
        assert bool(torch.isfinite(a).all()), name
        assert relative(a, b.transpose(1, 2)) <= 1e-4, name
    assert not any(bool(t[1].any()) for t in got)


@pytest.mark.parametrize("kind", ["trainable", "frozen", "autocast", "autocast transposed", "frozen autocast"])
def test_saved_act8_leaves_weights(kind):
    """the input's gradient needs the weight and not the input: bit for bit that of the plain run.  (A frozen weight's autocast copy has no graph that leads to the
    weight: there the context is told)"""
    from movedepth_amd import ops

    torch.manual_seed(0)
    m = torch.nn.Linear(1024, 1024, bias=False).cuda()
    f = (lambda t: t @ m.weight) if kind == "autocast transposed" else m
    if kind.startswith("frozen"):
        m.weight.requires_grad_(False)
    g = gen(4)
    x, go = randn(g, 2048, 1024).requires_grad_(), randn(g, 2048, 1024)

    def run():
        with torch.autocast("cuda", torch.bfloat16, enabled="autocast" in kind):
            return f(x * 1.0)

    y = run()
    want, = torch.autograd.grad(y, x, go.to(y.dtype))
    with ops.saved_act8(weights=m.parameters()) if kind == "frozen autocast" else ops.saved_act8():
        y = run()
    got, = torch.autograd.grad(y, x, go.to(y.dtype))
    assert torch.equal(got, want)


# --------------------------------------------------------------------------- scores of minus infinity, values beyond the pieces
def masked_reference(q, k, v, out, scale, go):
    """the definition without the keys `out`, whose weight is 0"""
    mask = torch.ones(k.shape[:2], dtype=torch.bool)
    mask[:, out] = False
    return ref.cross_attention(q, k, v, mask, scale, go)


PLACES = {"first": [0], "first tile": list(range(40)), "a later tile": [70, 71, 130], "last": [149], "most": list(range(3, 150))}


@pytest.mark.parametrize("Nq", [1, 40, 300])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("place", PLACES)
def test_a_score_of_minus_infinity_has_weight_zero(place, dtype, Nq):
    """every query's first element is 1 or 2, some keys' -inf: those scores are -inf and their weights 0, whichever key comes first.  The gradient of q's first
    element multiplies that weight with the infinity and is left out; the keys' own gradients are 0"""
    g, dt = gen(5), DT[dtype]
    q, go = randn(g, 2, Nq, 2, 32, dtype=dt), randn(g, 2, Nq, 2, 32, dtype=dt)
    k, v = randn(g, 2, 150, 2, 32, dtype=dt), randn(g, 2, 150, 2, 32, dtype=dt)
    q[..., 0] = torch.randint(1, 3, q.shape[:3], generator=g).to(dt).cuda()
    out = PLACES[place]
    want = masked_reference(q, k, v, out, 0.2, go)
    vals = want["dv"]
    want["dv"] = (vals[0], vals[1] + ref.tiny_of(dt))
    k[:, out, :, 0] = float("-inf")
    got = base.run_attention(q, k, v, None, 0.2, go)
    ref.within(got["o"], *want["o"], "o")
    ref.within(got["dq"][..., 1:], want["dq"][0][..., 1:], want["dq"][1][..., 1:], "dq")
    for name in ("dk", "dv"):
        ref.within(got[name], *want[name], name)


@pytest.mark.parametrize("Nq", [1, 50])
@pytest.mark.parametrize("dtype", DT)
def test_every_score_of_minus_infinity(dtype, Nq):
    """no key with a weight: zeros and no gradients, as for a query whose keys are all masked"""
    g, dt = gen(6), DT[dtype]
    q, go = randn(g, 1, Nq, 1, 16, dtype=dt), randn(g, 1, Nq, 1, 16, dtype=dt)
    k, v = randn(g, 1, 90, 1, 16, dtype=dt), randn(g, 1, 90, 1, 16, dtype=dt)
    q[..., 0] = 1
    k[..., 0] = float("-inf")
    got = base.run_attention(q, k, v, None, 0.2, go)
    for name in ("o", "dk", "dv"):
        assert not bool(got[name].any()), name
    assert not bool(got["dq"][..., 1:].any())


@pytest.mark.parametrize("Nq", [1, 40, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_beyond_the_range_below(dtype, Nq):
    """finite rows whose product passes the range of 32 bits below (-1e38 and less): weight 0, and gradients as without those keys"""
    g, dt = gen(7), DT[dtype]
    q, go = randn(g, 2, Nq, 2, 32, dtype=dt), randn(g, 2, Nq, 2, 32, dtype=dt)
    k, v = randn(g, 2, 150, 2, 32, dtype=dt), randn(g, 2, 150, 2, 32, dtype=dt)
    out = [0, 1, 35, 149]
    q[..., 0], k[..., 0] = 1e25, 0
    want = masked_reference(q, k, v, out, 0.2, go)
    k[:, out, :, 0] = -1e20
    got = base.run_attention(q, k, v, None, 0.2, go)
    for name in ("o", "dk", "dv"):
        ref.within(got[name], *want[name], name)
    # 0 times -1e20 is 0; but the sums' own rounding in front of it is not of the other keys' size
    ref.within(got["dq"][..., 1:], want["dq"][0][..., 1:], want["dq"][1][..., 1:], "dq")
    assert bool(torch.isfinite(got["dq"]).all())


@pytest.mark.parametrize("Nq", [2, 40])
@pytest.mark.parametrize("size", [1e12, 1e20, 3.3e38])
def test_float32_values_beyond_the_pieces(size, Nq):
    """large q against small k and the other way round, and large v and g: the products are ordinary numbers whatever the operands' own size.  Gradients of the small
    ones can fall below the normal range, where each of a sum's additions is off by up to half of the smallest step, 2^-150"""

    def check(got, want, what):
        base.check(got, {n: (val, tol + (70 + 2 * Nq) * 2.0 ** -150) for n, (val, tol) in want.items()}, what)

    g = gen(8)
    q, go = randn(g, 2, Nq, 2, 24), randn(g, 2, Nq, 2, 24)
    k, v = randn(g, 2, 70, 2, 24), randn(g, 2, 70, 2, 24)
    mask = base.make_mask("random", 2, 70, g)
    big = (q / q.abs().max()).sign() * size
    gq = go / 1e3 if Nq > 2 else go                          # (40 rows of 3.3e38: dk would be up to 9.2e38, which float32 does not hold)
    check(base.run_attention(big, k / size, v, mask, 0.3, gq), ref.cross_attention(big, k / size, v, mask, 0.3, gq), "large q")
    big = torch.where(k > 0, size, -size)
    check(base.run_attention(q / size, big, v, mask, 0.3, go / 1e3), ref.cross_attention(q / size, big, v, mask, 0.3, go / 1e3), "large k")
    big = torch.where(v > 0, size, -size) / 4
    check(base.run_attention(q, k, big, mask, 0.3, go / size), ref.cross_attention(q, k, big, mask, 0.3, go / size), "large v")
    if size < 1e30:
        check(base.run_attention(q, k, v / size, mask, 0.3, go * size), ref.cross_attention(q, k, v / size, mask, 0.3, go * size), "large g")


@pytest.mark.parametrize("need", ["qkv", "q", "kv"])
@pytest.mark.parametrize("d", [7, 40, 100])
def test_float32_rows_beyond_the_pieces_in_every_layout(d, need):
    """shared key heads, views of a joint projection, a mask with a sequence without keys, an expanded gradient, some of the gradients only; one sequence holds the large rows,
    and the others have the bits that they have without it"""
    from movedepth_amd import ops

    g = gen(15)
    q = randn(g, 3, 6, 50, d).transpose(1, 2)
    kv = randn(g, 3, 130, 2, 2, d)
    mask = (torch.rand(3, 130, generator=g) < 0.7).cuda()
    mask[1] = False
    go = randn(g, 1, 50, 6, 1).expand(3, 50, 6, d)

    def run():
        ts = {"q": q, "k": kv[:, :, 0], "v": kv[:, :, 1]}
        ts = {n: t.detach().requires_grad_(n in need) for n, t in ts.items()}
        o = ops.cross_attention(**ts, key_mask=mask, scale=0.2)
        names = [n for n in ts if n in need]
        return dict(zip(["o"] + ["d" + n for n in names], [o.detach(), *torch.autograd.grad(o, [ts[n] for n in names], go)]))

    plain = run()
    kv[2, 3, 0, :, 0], mask[2, 3], q[2, ..., 0] = float("-inf"), True, 1.5
    seen = mask.clone()
    seen[2, 3] = False
    got, want = run(), ref.cross_attention(q, kv[:, :, 0], kv[:, :, 1], seen, 0.2, go)
    for n in got:
        assert torch.equal(got[n][:2], plain[n][:2]), n
        skip = 1 if n == "dq" else 0                              # (its first element is a weight of 0 times -inf)
        ref.within(got[n][..., skip:], want[n][0][..., skip:], want[n][1][..., skip:], n)


@pytest.mark.parametrize("Nq", [1, 40])
@pytest.mark.parametrize("dtype", DT)
def test_an_infinite_value_reaches_its_own_column(dtype, Nq):
    """v = inf under a positive weight: that element of every output is inf, the others are what they were; a NaN query stays in its own row"""
    from movedepth_amd import ops

    g, dt = gen(9), DT[dtype]
    q, k, v = randn(g, 1, Nq, 1, 32, dtype=dt), randn(g, 1, 60, 1, 32, dtype=dt), randn(g, 1, 60, 1, 32, dtype=dt)
    want = ref.cross_attention(q, k, v, None, 0.1)["o"]
    v[0, 33, 0, 5] = float("inf")
    with torch.no_grad():
        o = ops.cross_attention(q, k, v, None, 0.1)
        assert bool((o[..., 5] == float("inf")).all())
        keep = [i for i in range(32) if i != 5]
        ref.within(o[..., keep], want[0][..., keep], want[1][..., keep], "o")
        if Nq > 1:
            q[0, 7, 0, 3] = float("nan")
            o = ops.cross_attention(q, k, v, None, 0.1)
            rows = [i for i in range(Nq) if i != 7]
            assert bool(torch.isnan(o[0, 7]).all())
            ref.within(o[:, rows][..., keep], want[0][:, rows][..., keep], want[1][:, rows][..., keep], "o")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_the_bound_on_the_scores_holds_at_its_ends(dtype):
    """rows so small that their squares vanish, against large keys and a large scale: the scores are in the hundreds; and weights of 2^45 times values of 1e28, whose
    sums pass the range unless the running maximum is taken off"""
    from movedepth_amd import ops

    g, dt = gen(10), DT[dtype]
    q = (randn(g, 1, 64, 1, 16).sign() * 5e-24).to(dt)
    k, v = (randn(g, 1, 200, 1, 16) * 1e18).to(dt), randn(g, 1, 200, 1, 16, dtype=dt)
    with torch.no_grad():
        ref.within(ops.cross_attention(q, k, v, None, 1e7), *ref.cross_attention(q, k, v, None, 1e7)["o"], "small rows")
        q, k = torch.full((1, 64, 1, 16), 1.4, device="cuda", dtype=dt), torch.full((1, 200, 1, 16), 1.4, device="cuda", dtype=dt)
        v = (randn(g, 1, 200, 1, 16) + 3).to(dt) * 1e28
        ref.within(ops.cross_attention(q, k, v, None, 1.0), *ref.cross_attention(q, k, v, None, 1.0)["o"], "large values")


@pytest.mark.parametrize("qscale", [0.3, 20.0])
@pytest.mark.parametrize("Nq", [2, 40, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sums_of_large_values_stay_in_range(dtype, Nq, qscale):
    """values near the range's end: any number of them weighs no more than one, though their plain sum passes the range"""
    from movedepth_amd import ops

    g, dt = gen(13), DT[dtype]
    q, k = randn(g, 1, Nq, 2, 16, dtype=dt, scale=qscale), randn(g, 1, 4000, 2, 16, dtype=dt)
    v = (randn(g, 1, 4000, 2, 16).sign() * 0.5 + 1).to(dt) * 2.0 ** 126
    with torch.no_grad():
        ref.within(ops.cross_attention(q, k, v, None, 1.0), *ref.cross_attention(q, k, v, None, 1.0)["o"], "o")


# --------------------------------------------------------------------------- float16 gradients of different sizes
@pytest.mark.parametrize("kind", ["sequences", "rows", "heads"])
def test_cross_attention_float16_gradients_of_different_sizes(kind):
    """one half of the gradient is 1e6 times the other: the small half's results are as exact as the large one's.  Norm-wise against 64 bits: dS and the result are each
    rounded to the type once, and o, which D is formed from; 2^-11 each at most, taken four times for the elements near zero"""
    g = gen(11)
    q, go = randn(g, 2, 64, 2, 64, dtype=torch.float16), randn(g, 2, 64, 2, 64)
    k, v = randn(g, 2, 1024, 2, 64, dtype=torch.float16), randn(g, 2, 1024, 2, 64, dtype=torch.float16)
    part = {"sequences": (slice(1, 2),), "rows": (slice(None), slice(1, None, 2)), "heads": (slice(None), slice(None), slice(1, 2))}[kind]
    size = torch.full_like(go, 8e3)
    size[part] = 8e-3
    go = (go * size).half()
    got, want = base.run_attention(q, k, v, None, 0.125, go), ref.cross_attention(q, k, v, None, 0.125, go)
    for name in ("dq",) if kind == "rows" else ("dq", "dk", "dv"):
        assert relative(got[name][part], want[name][0][part]) <= 4 * ref.u_of(torch.float16), name
    for name in ("dq", "dk", "dv"):
        assert relative(got[name], want[name][0]) <= 4 * ref.u_of(torch.float16), name


# --------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("C", [8, 48, 96, 777, 2056, 3000, 5000])
def test_layer_norm_of_rows_without_deviation(C):
    """a constant row is its own mean: y is b however far from zero it lies.  The mean's error, at most k = C / 64 + 24 roundings of the sum and the division's, is
    itself found as the mean of the deviations, off by as many roundings of it, and multiplied by 1 / sqrt(eps)"""
    from movedepth_amd import ops

    g = gen(12)
    x = torch.tensor([0.0, 3.0, 1000.1, -12345.678, 3.3e5, 1.7e6], device="cuda")[:, None].expand(6, C).contiguous().requires_grad_()
    w, b, go = randn(g, C), randn(g, C), randn(g, 6, C)
    y = ops.layer_norm(x, w, b)
    k = (C / 64 + 26) * ref.U32
    tol = w.abs().double().cpu() * x.detach().abs().double().cpu() * k * k * 1e-5 ** -0.5 + 4 * ref.U32 * b.abs().double().cpu()
    ref.within(y, b.double().cpu().expand(6, C), tol, "y")
    dx, = torch.autograd.grad(y, x, go)
    h = (go * w).double().cpu()
    want = (h - h.mean(1, keepdim=True)) * 1e-5 ** -0.5
    assert relative(dx, want) <= 1e-5


@pytest.mark.parametrize("act_bits", [0, 8])
@pytest.mark.parametrize("C", [24, 777, 3000, 5000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_layer_norm_keeps_what_is_not_finite_in_its_row(bad, C, act_bits):
    g = gen(14)
    x, w, b, go = randn(g, 9, C), randn(g, C), randn(g, C), randn(g, 9, C)
    rows = [i for i in range(9) if i != 4]
    want = ref.layer_norm(x[rows], w, b, 1e-5, go[rows], act_bits)
    x[4, C // 2] = bad
    got = base.run_layer_norm(x, w, b, 1e-5, go, act_bits)
    assert bool(torch.isnan(got["y"][4]).all()) and bool(torch.isnan(got["dx"][4]).all()) and bool(torch.isnan(got["dw"]).all())
    check({n: got[n][rows] for n in ("y", "dx")}, {n: want[n] for n in ("y", "dx")}, "the other rows")
    assert bool(torch.isfinite(got["db"]).all())


# --------------------------------------------------------------------------- forward mode
def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as fw

    from movedepth_amd import ops

    x = torch.ones(4, 16, device="cuda")
    t = torch.ones(1, 4, 1, 16, device="cuda")
    for no_grad in (False, True):
        with fw.dual_level(), torch.set_grad_enabled(not no_grad):
            for call in (lambda: ops.layer_norm(fw.make_dual(x, x)), lambda: ops.layer_norm(x, fw.make_dual(x[0], x[0])), lambda: ops.cross_attention(fw.make_dual(t, t), t, t),
                         lambda: ops.cross_attention(t, t, fw.make_dual(t, t))):
                with pytest.raises(RuntimeError):
                    call()
            ops.layer_norm(x)


# --------------------------------------------------------------------------- sizes of the framework's own mixed-precision path
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("kind", ["none", "random"])
def test_cross_attention_small_heads_in_two_bytes(kind, dtype):
    """two heads of 16 over thousands of tokens"""
    base.attention_case(1, 500, 5120, 2, 2, 16, dtype, kind)
    base.attention_case(1, 2500, 300, 2, 2, 16, dtype, kind)


# --------------------------------------------------------------------------- the trainer
def test_the_erased_region_does_not_come_back_through_the_other_frames(monkeypatch):
    """--match_attention: in the pass whose reference image has a rectangle erased nothing may depend on what stood there; both sides of its cost volume are compared
    between two images that differ in the rectangle only.  The encoder's library normalisation sums in an order that changes from run to run (the same image
    twice, without any attention: 6e-7 of 2), so 32-bit rounding through its layers, 1e-4 of the largest, is allowed; what leaks in is of the features' size"""
    from movedepth_amd import ops, synthetic, trainer

    monkeypatch.setattr(trainer, "random_image_mask", lambda img, size: erase(img))
    keep = {}

    def erase(img):
        m = torch.ones_like(img)
        m[:, :, 10:31, 20:62] = 0
        return img * m, m

    calls, real = [], ops.costvol_grouped

    def record(ref_feat, src_feat, *a, **kw):
        calls.append((ref_feat.detach().clone(), src_feat.detach().clone()))
        return real(ref_feat, src_feat, *a, **kw)

    monkeypatch.setattr(ops, "costvol_grouped", record)
    make = synthetic.make_inputs
    _, _, t = base.step(["--match_attention", "2"])
    torch.nn.init.normal_(t.models["match_attn"].out.weight, std=0.5)
    state = {n: {k: v.clone() for k, v in m.state_dict().items()} for n, m in t.models.items()}

    def changed(*a, **kw):
        inputs = make(*a, **kw)
        inputs["color_aug", 0, 0] = inputs["color_aug", 0, 0].clone()
        inputs["color_aug", 0, 0][:, :, 10:31, 20:62] = 0.9
        return inputs

    for name, inputs in (("plain", make), ("changed", changed)):
        calls.clear()
        monkeypatch.setattr(synthetic, "make_inputs", inputs)
        base.step(["--match_attention", "2"], models=state)
        keep[name] = list(calls)
    n = len(keep["plain"]) // 2
    assert n >= 1 and len(keep["changed"]) == 2 * n
    r0, r1 = keep["plain"][0][0], keep["changed"][0][0]
    assert float((r0 - r1).abs().max()) > 0.1 * float(r0.abs().max())          # the first pass sees the difference
    for (r0, s0), (r1, s1) in zip(keep["plain"][n:], keep["changed"][n:]):
        assert float((r0 - r1).abs().max()) <= 1e-4 * float(r0.abs().max()) and float((s0 - s1).abs().max()) <= 1e-4 * float(s0.abs().max())


def eight_bits(t):
    """t through 8 bits in the order of its storage, in torch operations on whole groups (definition: 32 neighbours, the least power of two that leaves the largest at
    127 or below)"""
    flat = t.detach().as_strided((t.numel(),), (1,), t.storage_offset()).double()
    part = torch.nn.functional.pad(flat, (0, -t.numel() % 32)).view(-1, 32)
    mant, ex = torch.frexp(part.abs().amax(1, keepdim=True))
    step = torch.ldexp(torch.ones_like(mant), (ex - 7 + (mant * 128 >= 127.5).int()).clamp(-126, 121))
    out = torch.empty_strided(t.shape, t.stride(), device=t.device, dtype=t.dtype)
    out.as_strided((t.numel(),), (1,)).copy_((torch.round(part / step).clamp(-127, 127) * step).view(-1)[:t.numel()])
    return out


def test_trainer_keeps_the_regularisers_activations_in_8_bits(monkeypatch):
    """--act_bits 8: the gradients of all that the regulariser's backward pass reaches are those of a run that keeps its activations as 8-bit values made by torch
    operations, and not the plain step's.  The activations of two runs differ by about 2e-6 of their largest (library sums in an order that changes), so one in
    2e-6 * 127.5 = 2.5e-4 rounds to the next 8-bit step, 1 / 64 of its group's largest, at most sqrt(32) / 64 of the root mean square: sqrt(2.5e-4) * 0.09 = 1.4e-3
    norm-wise; where that step is the one next to zero (2 of 127) a ReLU lets a gradient pass or not: sqrt(2.5e-4 * 2 / 127) = 2e-3.  Together below 5e-3; a
    wrong stride would be off by the gradient's whole size"""
    from movedepth_amd import ops

    real_context, real_pack, packed, by_hand = ops.saved_act8, ops.act8_pack, [], []
    limit = 4096

    def pack(t):
        packed.append(t.numel())
        return real_pack(t)

    def by_torch(weights=(), **kw):
        own = {w.data_ptr() for w in weights}

        def save(t):
            if t.dtype != torch.float32 or t.numel() < limit or t.data_ptr() in own or not ops._is_dense(t):
                return t.detach()
            by_hand.append(t.numel())
            return eight_bits(t)

        return torch.autograd.graph.saved_tensors_hooks(save, lambda t: t)

    _, _, t = base.step(["--match_attention", "2"])
    torch.nn.init.normal_(t.models["match_attn"].out.weight, std=0.2)
    state = {n: m.state_dict() for n, m in t.models.items()}
    _, plain, _ = base.step(["--match_attention", "2"], models=state)
    args = ["--match_attention", "2", "--act_bits", "8"]
    monkeypatch.setattr(ops, "act8_pack", pack)
    monkeypatch.setattr(ops, "saved_act8", lambda min_numel=None, **kw: real_context(min_numel=limit, **kw))
    _, got, _ = base.step(args, models=state)
    assert len(packed) >= 20 and max(packed) >= 2 * 16 * 16 * 16 * 32          # two passes through the regulariser
    monkeypatch.setattr(ops, "saved_act8", by_torch)
    _, want, _ = base.step(args, models=state)
    assert packed == by_hand                                  # the same tensors in the same order
    names = [n for n in want if n.split(".")[0] in ("reg3d", "mvs_encoder", "match_attn") and want[n] is not None and bool(want[n].any())]
    assert len([n for n in names if n.startswith("reg3d")]) >= 10
    for n in names:
        assert relative(got[n], want[n]) <= 5e-3, n
    # the last layer's weight gradient is a sum over rounded activations, nothing behind it is: off by the rounding, at most half a step = 1 / 127.5 of the largest
    # of 32 neighbours, which is at most sqrt(32) times their root mean square
    off = [relative(r["reg3d.prob.weight"], plain["reg3d.prob.weight"]) for r in (got, want)]
    print("last layer's weight gradient off by %.3g, by %.3g with torch's 8 bits" % tuple(off))
    assert 10 * relative(got["reg3d.prob.weight"], want["reg3d.prob.weight"]) < min(off) and max(off) <= 32 ** 0.5 / 127.5
