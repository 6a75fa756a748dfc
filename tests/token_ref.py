"""Definitions in 64 bits of the token operators (layer norm, 8-bit activations, cross attention) with, beside each result, a bound on what a
kernel that rounds as documented may be off by: every element's bound follows from the roundings (u = half a step of the type, 2^-24 for each
32-bit operation) and the sizes of the terms, none from a measurement."""
import torch

U32 = 2.0 ** -24


def u_of(dtype):
    return torch.finfo(dtype).eps / 2


def tiny_of(dtype):
    """half the smallest step near zero: what a result below the normal range may lose"""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def within(got, want, tol, what):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, "%s: shape %s, not %s" % (what, tuple(got.shape), tuple(want.shape))
    assert bool(torch.isfinite(got).all()), "%s: not finite" % what
    off = (got - want).abs()
    bad = off > tol
    if bool(bad.any()):
        r = torch.where(tol > 0, off / tol, torch.where(off > 0, float("inf"), 0.0))
        i = int(r.argmax())
        raise AssertionError("%s: %d of %d off by more than the bound, the worst %.3g against %.3g (value %.6g)" % (
            what, int(bad.sum()), bad.numel(), float(off.flatten()[i]), float(tol.flatten()[i]), float(want.flatten()[i])))


# --------------------------------------------------------------------------- 8-bit activations
RANGE = {torch.float32: (-126, 121), torch.bfloat16: (-126, 121), torch.float16: (-24, 9)}


def act8(x):
    """(rows, C) of any of the types -> the same in float64, through 8 bits: group by group, from the definition"""
    lo, hi = RANGE[x.dtype]
    y = x.detach().double().cpu().clone()
    rows, C = y.shape
    for r in range(rows):
        for c in range(0, C, 32):
            part = y[r, c:c + 32]
            if not bool(torch.isfinite(part).all()):
                part[:] = float("nan")
                continue
            a, e = float(part.abs().max()), lo
            while e < hi and round(a / 2.0 ** e) > 127:      # (Python rounds ties to even)
                e += 1
            part[:] = torch.clamp(torch.round(part / 2.0 ** e), -127, 127) * 2.0 ** e
    return y


# --------------------------------------------------------------------------- layer norm
def layer_norm(x, w, b, eps, g=None, act_bits=0):
    """x (rows, C).  -> {name: (value, bound)} for y and, with g, dx, dw, db"""
    u, tiny = u_of(x.dtype), tiny_of(x.dtype)
    x8 = act8(x) if act_bits else None
    x, (rows, C) = x.detach().double().cpu(), x.shape
    w = torch.ones(C, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(1, keepdim=True)
    var = (x - mean).square().mean(1, keepdim=True)
    r = (var + eps).rsqrt()
    n = (x - mean) * r
    # sums over a row: at most C / 64 + 24 additions behind each other, each off by U32 of the terms' magnitudes
    k = (C / 64 + 24) * U32
    off_mean = k * x.abs().mean(1, keepdim=True) + U32 * x.abs().amax(1, keepdim=True)
    # of the variance: its own sum, and what the mean's error adds (the deviations' sum is zero, so its square only, bounded by it all the same)
    off_r = r * (k + (off_mean * r).square() + 2 * off_mean * r * U32 * C ** 0.5)
    off_n = off_mean * r + (x - mean).abs() * off_r + 4 * U32 * n.abs()
    y = n * w + b
    out = {"y": (y, u * y.abs() + tiny + w.abs() * off_n + 4 * U32 * ((n * w).abs() + b.abs()))}
    if g is None:
        return out
    g = g.detach().double().cpu()
    if x8 is not None:
        n = (x8 - mean) * r
        off_n = off_mean * r + (x8 - mean).abs() * off_r + 4 * U32 * n.abs()
    h = g * w
    mh, mhn = h.mean(1, keepdim=True), (h * n).mean(1, keepdim=True)
    off_mh = k * h.abs().mean(1, keepdim=True)
    off_mhn = k * (h * n).abs().mean(1, keepdim=True) + (h.abs() * off_n).mean(1, keepdim=True)
    inner = h - mh - n * mhn
    off = off_mh + off_n * mhn.abs() + n.abs() * off_mhn + 8 * U32 * (h.abs() + mh.abs() + (n * mhn).abs())
    out["dx"] = (r * inner, u * (r * inner).abs() + tiny + r * off + inner.abs() * off_r)
    # sums over the rows: at most rows / 64 + 64 additions behind each other
    k = (rows / 64 + 64) * U32
    out["dw"] = ((g * n).sum(0), k * (g * n).abs().sum(0) + (g.abs() * off_n).sum(0))
    out["db"] = (g.sum(0), k * g.abs().sum(0))
    return out


# --------------------------------------------------------------------------- cross attention
def cross_attention(q, k, v, mask, scale, g=None):
    """q (B, Nq, Hq, d), k, v (B, Nk, Hk, d), mask (B, Nk) bool or None -> {name: (value, bound)} for o and, with g, dq, dk, dv"""
    dt = q.dtype
    u, tiny = u_of(dt), tiny_of(dt)
    up = 0.0 if dt == torch.float32 else u              # softmax weights (and dS) are rounded to 2-byte types before their products
    B, Nq, Hq, d = q.shape
    Nk, Hk = k.shape[1:3]
    G = Hq // Hk
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    if mask is not None:
        m = mask.cpu()[:, :, None, None]
        k, v = (torch.where(m, t, torch.zeros((), dtype=torch.float64)) for t in (k, v))
    qh, kh, vh = q.transpose(1, 2), k.repeat_interleave(G, 2).transpose(1, 2), v.repeat_interleave(G, 2).transpose(1, 2)   # (B, H, N, d)
    s = qh @ kh.transpose(2, 3) * scale
    # products of d terms, the scaling, and 2^x of a 32-bit argument; also what the lowest of three bf16 pieces of a 32-bit operand leaves out
    off_s = (d + 16) * U32 * abs(scale) * (qh.abs() @ kh.abs().transpose(2, 3))
    if mask is not None:
        s = s.masked_fill(~mask.cpu()[:, None, None, :], float("-inf"))
    if Nk:
        top = s.amax(3, keepdim=True)
        p = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        l = p.sum(3, keepdim=True)
        p = p / torch.where(l > 0, l, torch.ones_like(l))
    else:
        p = s
    # relative error of a normalised weight: its own exponent, the denominator's (a mean of the same errors), the sums behind each other.
    # exp(x) for x in [-off, off] is within e^off - 1; weights below 2^-126 of the largest may vanish
    es = torch.expm1(off_s.amax(3, keepdim=True) if Nk else off_s.new_zeros(B, Hq, Nq, 1)) * 2 + (Nk + 16) * U32
    ep = es + up
    A = p @ vh.abs()
    o = p @ vh
    # a 32-bit weight below 2^-126 is subnormal or gone, a 2-byte one loses up to half its type's smallest step
    gone = 2.0 ** -125
    small = (tiny if up else 0.0) + gone
    off_o = ep * A + small * vh.abs().sum(2, keepdim=True)

    def back(t):
        return t.transpose(1, 2).contiguous()

    out = {"o": (back(o), back(u * o.abs() + tiny + off_o))}
    if g is None:
        return out
    gh = g.detach().double().cpu().transpose(1, 2)
    dp = gh @ vh.transpose(2, 3)
    D = (gh * o).sum(3, keepdim=True)
    off_dp = (d + 16) * U32 * (gh.abs() @ vh.abs().transpose(2, 3))
    off_D = (gh.abs() * (u * o.abs() + tiny + off_o)).sum(3, keepdim=True) + (d + 16) * U32 * (gh * o).abs().sum(3, keepdim=True)
    ds = p * (dp - D)
    # p is rounded for dv only; ds is rounded once; both carry the exponent's error
    off_ds = ds.abs() * (ep + 4 * U32) + p * (1 + es) * (off_dp + off_D + 4 * U32 * (dp.abs() + D.abs())) + gone * (dp.abs() + D.abs())

    def shared(t):                                       # sum over the query heads of one key head
        return t.reshape(B, Hk, G, Nk, d).sum(2)

    dq = scale * (ds @ kh)
    off_dq = abs(scale) * (off_ds @ kh.abs() + (Nk + 16) * U32 * (ds.abs() @ kh.abs()) + small * kh.abs().sum(2, keepdim=True))
    out["dq"] = (back(dq), back(u * dq.abs() + tiny + off_dq))
    chain = (Nq * G + 16) * U32
    dk = shared(scale * (ds.transpose(2, 3) @ qh))
    off_dk = shared(abs(scale) * (off_ds.transpose(2, 3) @ qh.abs() + chain * (ds.abs().transpose(2, 3) @ qh.abs())
                                  + small * qh.abs().sum(2, keepdim=True)))
    dv = shared(p.transpose(2, 3) @ gh)
    off_dv = shared((p * ep + chain * p).transpose(2, 3) @ gh.abs() + small * gh.abs().sum(2, keepdim=True))
    out["dk"] = (back(dk), back(u * dk.abs() + tiny + off_dk))
    out["dv"] = (back(dv), back(u * dv.abs() + tiny + off_dv))
    if mask is not None:
        for name in ("dk", "dv"):
            val, tol = out[name]
            out[name] = (torch.where(m, val, torch.zeros_like(val)), torch.where(m, tol, torch.zeros_like(tol)))
    return out
