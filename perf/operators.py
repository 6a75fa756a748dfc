"""Cases of the framework's transformer operators: layer norm (ops.layer_norm), 8-bit activation checkpoints (ops.act8_pack / ops.act8_unpack
and layer_norm's act_bits=8) and attention from one frame's tokens to another's (ops.cross_attention).

`own = False` computes them in their plain form (elementary torch operations in 32 bits, rounded once at the end), `own = True` calls the
framework.  `exact` is the definition in 64 bits.  Shapes: a "token" is one pixel of the 1/4-resolution matching features -- 48 x 160 = 7680 tokens of
32 channels for a 192 x 640 image, 80 x 256 = 20480 of 64 for 320 x 1024 -- or generic where the case says so."""
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5
GROUP = 32                      # elements that share one power-of-two scale in the 8-bit format
SCALE_RANGE = {torch.float32: (-126, 121), torch.bfloat16: (-126, 121), torch.float16: (-24, 9)}   # exponents of that scale, by the type it stands for


def listed():
    return [
        # the latency of one small call: the tokens of a few queries, inference
        {"name": "ln_small_bf16", "op": "ln", "mode": "fwd", "dtype": "bf16", "rows": 8, "C": 512},
        # the matching features of a batch of 6 images of 192 x 640, fp32 training step
        {"name": "ln_match_f32", "op": "ln", "mode": "train", "dtype": "f32", "rows": 6 * 7680, "C": 32},
        # the same at 320 x 1024 under autocast, the input kept for the backward pass in 8 bits
        {"name": "ln_match8_bf16", "op": "ln", "mode": "train8", "dtype": "bf16", "rows": 6 * 20480, "C": 64},
        # odd sizes: rows that are not vectors of anything
        {"name": "ln_odd_f16", "op": "ln", "mode": "train", "dtype": "f16", "rows": 3001, "C": 777},
        # a wide model's rows (the last stage of the 50-layer encoder has 2048 channels)
        {"name": "ln_wide_bf16", "op": "ln", "mode": "train", "dtype": "bf16", "rows": 32768, "C": 2048},
        # the 3-D regulariser's full-resolution activation (6 x 16 x 96 x 48 x 160), stored for the backward pass and restored
        {"name": "act8_volume_f32", "op": "act8", "dtype": "f32", "n": 6 * 16 * 96 * 48 * 160},
        # a small odd activation
        {"name": "act8_odd_bf16", "op": "act8", "dtype": "bf16", "n": 1000003},
        # one query per sequence against a long encoder state with shared heads (serving)
        {"name": "xa_token_bf16", "op": "xa", "mode": "fwd", "dtype": "bf16", "B": 8, "Nq": 1, "Nk": 20480, "Hq": 16, "Hk": 4, "d": 64, "valid": 1.0, "empty": False},
        # reference-frame tokens to source-frame tokens, 192 x 640, batch 6, fp32 training step, source pixels partly masked
        {"name": "xa_match_f32", "op": "xa", "mode": "train", "dtype": "f32", "B": 6, "Nq": 7680, "Nk": 7680, "Hq": 2, "Hk": 2, "d": 16, "valid": 0.9, "empty": False},
        # the same at 320 x 1024 under autocast
        {"name": "xa_match_bf16", "op": "xa", "mode": "train", "dtype": "bf16", "B": 2, "Nq": 20480, "Nk": 20480, "Hq": 2, "Hk": 2, "d": 32, "valid": 1.0, "empty": False},
        # a ragged padded batch with shared heads, one sequence without a single valid key, inference
        {"name": "xa_ragged_f16", "op": "xa", "mode": "fwd", "dtype": "f16", "B": 3, "Nq": 1001, "Nk": 2777, "Hq": 8, "Hk": 2, "d": 128, "valid": 0.6, "empty": True},
        # a decoder's queries against an encoder's longer states, wide heads, training
        {"name": "xa_train_bf16", "op": "xa", "mode": "train", "dtype": "bf16", "B": 2, "Nq": 4096, "Nk": 8192, "Hq": 16, "Hk": 16, "d": 64, "valid": 1.0, "empty": False},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["ln", "ln", "act8", "xa", "xa", "xa"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "ln":
        C = _log(rng, 8, 4096)
        if rng.random() < 0.6:
            C = max(8, C // 8 * 8)
        return {"op": "ln", "mode": rng.choice(["fwd", "train", "train8"]), "dtype": dtype, "rows": _log(rng, 1, min(122880, 32768 * 1024 // C)), "C": C}
    if op == "act8":
        return {"op": "act8", "dtype": dtype, "n": _log(rng, 1000, 70000000)}
    d = rng.choice([8, 16, 24, 32, 40, 64, 80, 96, 128])
    Hk, G, B = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4]), rng.choice([1, 2, 3, 6])
    mode = rng.choice(["fwd", "train"])
    Nk = _log(rng, 1 if mode == "fwd" else 8, 20480)      # (a single key's weight is 1 whatever the inputs: the gradients of q and k are 0 there)
    most = int(1.6e9 * (16 if dtype == "f32" else 32) / (max(d, 32) * Hk * G * B * Nk))     # query rows that keep it cheaper than the listed ones
    return {"op": "xa", "mode": mode, "dtype": dtype, "B": B, "Nq": _log(rng, 1, max(1, min(8192, most))), "Nk": Nk, "Hq": Hk * G, "Hk": Hk, "d": d,
            "valid": rng.choice([1.0, 0.8, 0.5]), "empty": B > 1 and rng.random() < 0.3}


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0, shift=0.0):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] == "ln":
        train = case["mode"] != "fwd"
        s["x"] = randn(case["rows"], case["C"], scale=1.5, shift=0.3).requires_grad_(train)
        # parameters stay in 32 bits, as a module's under autocast
        s["w"] = randn(case["C"], dtype=torch.float32, scale=0.2, shift=1.0).requires_grad_(train)
        s["b"] = randn(case["C"], dtype=torch.float32, scale=0.2).requires_grad_(train)
        if train:
            s["g"] = randn(case["rows"], case["C"])
    elif case["op"] == "act8":
        s["x"] = torch.relu(randn(case["n"]))     # an activation: half of it zeros
    else:
        B, Nq, Nk, Hq, Hk, d = (case[k] for k in ("B", "Nq", "Nk", "Hq", "Hk", "d"))
        train = case["mode"] == "train"
        s["q"] = randn(B, Nq, Hq, d, scale=1.5).requires_grad_(train)
        s["k"] = randn(B, Nk, Hk, d).requires_grad_(train)
        s["v"] = randn(B, Nk, Hk, d).requires_grad_(train)
        if train:
            s["g"] = randn(B, Nq, Hq, d)
        s["mask"] = None
        if case["valid"] < 1 or case["empty"]:
            mask = torch.rand(B, Nk, device="cuda", generator=g) < case["valid"]
            if case["empty"]:
                mask[B - 1] = False
            s["mask"] = mask
    return s


# --------------------------------------------------------------------------- the operators
def run(state):
    case = state["case"]
    return {"ln": _run_ln, "act8": _run_act8, "xa": _run_xa}[case["op"]](state, case)


def _run_ln(s, case):
    x, w, b = s["x"], s["w"], s["b"]
    train, act8 = case["mode"] != "fwd", case["mode"] == "train8"
    if own:
        from movedepth_amd import ops
        if not train:
            with torch.no_grad():
                return {"y": ops.layer_norm(x, w, b, EPS)}
        y = ops.layer_norm(x, w, b, EPS, act_bits=8 if act8 else 0)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["g"])
        return {"y": y.detach(), "dx": dx, "dw": dw, "db": db}
    with torch.no_grad():
        xf = x.float()
        mean = xf.mean(1, keepdim=True)
        rstd = torch.rsqrt((xf - mean).square().mean(1, keepdim=True) + EPS)
        out = {"y": ((xf - mean) * rstd * w + b).to(x.dtype)}
        if train:
            if act8:
                xf = _through_8_bits(x).float()
            n, gf = (xf - mean) * rstd, s["g"].float()
            gw = gf * w
            out["dx"] = (rstd * (gw - gw.mean(1, keepdim=True) - n * (gw * n).mean(1, keepdim=True))).to(x.dtype)
            out["dw"], out["db"] = (gf * n).sum(0), gf.sum(0)
        return out


def _through_8_bits(x):
    """x (rows, C): what 8-bit whole numbers times a power of two per group of 32 neighbours in a row keep of it."""
    rows, C = x.shape
    lo, hi = SCALE_RANGE[x.dtype]
    f = torch.nn.functional.pad(x.detach().float(), (0, -C % GROUP)).view(rows, -1, GROUP)
    bits = f.abs().amax(2, keepdim=True).view(torch.int32)
    e = (((bits + 0x10000) >> 23) - 133).clamp(lo, hi)          # the least exponent that leaves the largest at 127 or below after rounding
    scale = ((e + 127) << 23).view(torch.float32)
    inv = ((127 - e) << 23).view(torch.float32)
    q = torch.round(f * inv).clamp(-127, 127)
    return (q * scale).view(rows, -1)[:, :C].to(x.dtype)


def _run_act8(s, case):
    if own:
        from movedepth_amd import ops
        return {"x": ops.act8_unpack(ops.act8_pack(s["x"]))}
    return {"x": _through_8_bits(s["x"].view(1, -1)).view(-1)}


def _by_head(t, Hk, dtype):
    """(B, N, H, d) -> (B * Hk, (H / Hk) * N, d): the query heads that share a key head behind each other"""
    B, N, H, d = t.shape
    return t.detach().to(dtype).view(B, N, Hk, H // Hk, d).permute(0, 2, 3, 1, 4).reshape(B * Hk, H // Hk * N, d)


def _from_head(t, like):
    B, N, H, d = like.shape
    Hk = t.shape[0] // B
    return t.view(B, Hk, H // Hk, N, d).permute(0, 3, 1, 2, 4).reshape(B, N, H, d).to(like.dtype)


def _run_xa(s, case):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        from movedepth_amd import ops
        if case["mode"] == "fwd":
            with torch.no_grad():
                return {"o": ops.cross_attention(q, k, v, key_mask=s["mask"])}
        o = ops.cross_attention(q, k, v, key_mask=s["mask"])
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["g"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    with torch.no_grad():
        Hk, scale = case["Hk"], case["d"] ** -0.5
        qf, kf, vf = _by_head(q, Hk, torch.float32), _by_head(k, Hk, torch.float32), _by_head(v, Hk, torch.float32)
        p = torch.bmm(qf, kf.transpose(1, 2).contiguous()).mul_(scale)
        if s["mask"] is not None:
            dead = ~s["mask"].repeat_interleave(Hk, 0)
            p.masked_fill_(dead[:, None, :], float("-inf"))
        p = p.sub_(p.amax(2, keepdim=True).clamp(min=-3e38)).exp_()
        p = p.div_(p.sum(2, keepdim=True).clamp(min=1e-30))        # a row without a valid key: all zeros
        of = torch.bmm(p, vf)
        out = {"o": _from_head(of, q)}
        if case["mode"] == "train":
            gf = _by_head(s["g"], Hk, torch.float32)
            out["dv"] = _from_head(torch.bmm(p.transpose(1, 2).contiguous(), gf), v)
            ds = torch.bmm(gf, vf.transpose(1, 2).contiguous()).sub_((gf * of).sum(2, keepdim=True)).mul_(p).mul_(scale)
            out["dq"] = _from_head(torch.bmm(ds, kf), q)
            out["dk"] = _from_head(torch.bmm(ds.transpose(1, 2).contiguous(), qf), k)
        return out


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "ln":
        n, train = case["rows"] * case["C"], case["mode"] != "fwd"
        return {"bytes": (4 if train else 2) * n * size + (4 if train else 2) * case["C"] * 4, "flops": (20 if train else 7) * n}
    if case["op"] == "act8":
        return {"bytes": 2 * case["n"] * size, "flops": 4 * case["n"]}
    B, Nq, Nk, Hq, Hk, d = (case[k] for k in ("B", "Nq", "Nk", "Hq", "Hk", "d"))
    train = case["mode"] == "train"
    live = (B - 1 if case["empty"] else B) * case["valid"]      # sequences' worth of keys that the mask leaves
    keys, queries = live * Nk * Hk * d * size, B * Nq * Hq * d * size
    masked = case["valid"] < 1 or case["empty"]
    # forward: q, k, v -> o; with the gradients also g -> dq, and dk, dv whole (zeros where masked).  Two products forward, five backward.
    return {"bytes": (2 * keys + 2 * queries) + (B * Nk if masked else 0) + (2 * queries + 2 * B * Nk * Hk * d * size if train else 0),
            "flops": (14 if train else 4) * live * Nq * Nk * Hq * d}


# --------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"ln": _exact_ln, "act8": _exact_act8, "xa": _exact_xa}[case["op"]](s, case)


def _round_8_bits(x, dtype):
    """x (rows, C) in 64 bits -> n * 2^e, n whole, |n| <= 127: e the least exponent of the type's range for which the group's largest value rounds to 127 or less (the range's last: cut off there)"""
    rows, C = x.shape
    lo, hi = SCALE_RANGE[dtype]
    parts = torch.cat([x, x.new_zeros(rows, -C % GROUP)], 1).reshape(rows, -1, GROUP)
    mant, ex = torch.frexp(parts.abs().max(2, keepdim=True).values)      # largest = mant * 2^ex, 1/2 <= mant < 1
    e = torch.clamp(ex - 7 + (mant * 128 >= 127.5).to(ex.dtype), lo, hi)
    step = ((e.long() + 1023) << 52).view(torch.float64)                 # 2^e from its bits: pow() is not exact, and half steps are ties
    return (torch.clamp(torch.round(parts / step), -127, 127) * step).reshape(rows, -1)[:, :C]


def _exact_act8(s, case):
    return {"x": _round_8_bits(s["x"].double()[None], s["x"].dtype)[0]}


def _exact_ln(s, case):
    x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
    var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
    sd = torch.sqrt(var + EPS)
    out = {"y": w * ((x - mean) / sd) + b}
    if case["mode"] != "fwd":
        if case["mode"] == "train8":
            x = _round_8_bits(x, s["x"].dtype)
        g, n, C = s["g"].double(), (x - mean) / sd, case["C"]
        out["db"], out["dw"] = g.sum(0), (g * n).sum(0)
        h = g * w
        out["dx"] = (h - h.sum(1, keepdim=True) / C - n * ((h * n).sum(1, keepdim=True) / C)) / sd
    return out


def _exact_xa(s, case):
    B, Nq, Nk, Hq, Hk, d = (case[k] for k in ("B", "Nq", "Nk", "Hq", "Hk", "d"))
    q, k, v = (s[n].double().transpose(1, 2) for n in ("q", "k", "v"))          # (B, H, N, d)
    G = Hq // Hk
    k, v = (t[:, :, None].expand(B, Hk, G, Nk, d).reshape(B, Hq, Nk, d) for t in (k, v))
    logits = torch.matmul(q, k.transpose(2, 3).contiguous()) / d ** 0.5
    if s["mask"] is not None:
        logits = torch.where(s["mask"][:, None, None, :], logits, -1e300)
    prob = torch.softmax(logits, 3)
    del logits
    if s["mask"] is not None:
        prob = prob * s["mask"][:, None, None, :]
    o = torch.matmul(prob, v)
    out = {"o": o.transpose(1, 2).contiguous()}
    if case["mode"] == "train":
        g = s["g"].double().transpose(1, 2)
        dv = torch.matmul(prob.transpose(2, 3).contiguous(), g.contiguous())
        dl = torch.matmul(g, v.transpose(2, 3).contiguous())
        dl = dl.sub_((dl * prob).sum(3, keepdim=True)).mul_(prob).div_(d ** 0.5)
        del prob
        dq, dk = torch.matmul(dl, k), torch.matmul(dl.transpose(2, 3).contiguous(), q.contiguous())
        dk, dv = (t.view(B, Hk, G, Nk, d).sum(2) for t in (dk, dv))
        out.update(dq=dq.transpose(1, 2).contiguous(), dk=dk.transpose(1, 2).contiguous(), dv=dv.transpose(1, 2).contiguous())
    return out
