"""64-bit definitions of qk_norm_rope, relative_attention and differential_attention with their gradients, and bounds on what a
kernel that computes in 32 bits and rounds its matrix operands to the inputs' type may be off by (test infrastructure).

Bounds, with u = eps / 2 of the type (one rounding) and e = 2^-24:
  scores   (d + 8) e sum |q||k| scale, and 4 e (|s| + log2 of the sums) for the exponent's own arithmetic: ds
  P        relative 2 ds (numerator and sum) before it is rounded
  out      u (sum P |v| + |out|) + 2 ds sum P |v|
  W        (dv + 8) e sum |dO||v|;  D: u sum |dO||o| (from the rounded output) + its 32-bit sum
  dS       2 ds |dS| + P (dW + dD) =: E, and u |dS| where it is a product's operand
  dq, dk   scale sum (E + u |dS|) |k| + u |dq|;  dv: u (sum P |dO| + |dv|) + 2 ds sum P |dO|
  dtable   sum of E over the bucket's pairs + n e sum |dS| + u |dtable|;  dlam alike without the last
fp16 rounds values below 2^-14 by 2^-25 absolutely (P at most, scaled to a row maximum of one at least)."""
import math

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seen(B, Tq, Tk, causal, lens, start):
    """(B, Tq, Tk) truth values and relative positions"""
    i, j = torch.arange(Tq)[None, :, None], torch.arange(Tk)[None, None, :]
    st = (torch.full((B,), Tk - Tq) if start is None else start.cpu().long())[:, None, None]
    rel = j - (st + i)
    ok = torch.ones((B, Tq, Tk), dtype=torch.bool)
    if causal:
        ok &= rel <= 0
    if lens is not None:
        ok &= j < lens.cpu().long().clamp(0, Tk)[:, None, None]
    return ok, rel


def attention(maps, q, k, v, causal=False, scale=None, lens=None, start=None, table=None, buckets=None, lam=None, dout=None):
    """{name: (value, bound)}; all tensors on the CPU, layouts as the framework's"""
    dt = q.dtype
    u = half_step(dt)
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    B, Tq, _, d = q.shape
    Tk, Hkv = v.shape[1:3]
    H = q.shape[2] // maps
    G = H // Hkv
    scale = d ** -0.5 if scale is None else scale
    ok, rel = seen(B, Tq, Tk, causal, lens, start)
    live = torch.arange(Tk)[None, :] < (torch.full((B,), Tk) if lens is None else lens.cpu().long().clamp(0, Tk))[:, None]
    zero = ~live[:, :, None, None]
    q, k, v = q.double(), k.double().masked_fill(zero, 0.0), v.double().masked_fill(zero, 0.0)   # behind the length: never used
    kk, vv = k.repeat_interleave(G, 2) if maps == 1 else k.unflatten(2, (Hkv, 2)).repeat_interleave(G, 2).flatten(2, 3), v.repeat_interleave(G, 2)
    ok4 = ok[:, None]
    P, dS_s = [], []
    lse = torch.zeros((B, H * maps, Tq), dtype=torch.float64)
    for m in range(maps):
        qm, km = q[:, :, m::maps].transpose(1, 2), kk[:, :, m::maps].transpose(1, 2)
        s = torch.matmul(qm, km.transpose(2, 3)) * scale
        es = (d + 8) * E * scale * torch.matmul(qm.abs(), km.abs().transpose(2, 3))
        if table is not None:
            R = buckets.shape[0] // 2
            s = s + table.double()[:, buckets.long()[rel.clamp(-R, R) + R]].transpose(0, 1)
        s = s.masked_fill(~ok4, -math.inf)
        mx = s.amax(-1, keepdim=True)
        mx = torch.where(mx == -math.inf, 0.0, mx)
        p = torch.exp(s - mx)
        tot = p.sum(-1, keepdim=True)
        lse[:, m::maps] = (mx + tot.log()).squeeze(-1)
        P.append(p / tot.clamp_min(1e-300))
        fin = torch.where(torch.isfinite(s), s.abs(), 0.0)
        e = torch.where(ok4, es, 0.0).amax(-1, keepdim=True) + 4 * E * (fin.amax(-1, keepdim=True) + math.log2(Tk + 1) + 8)
        dS_s.append(e)
    vt = vv.transpose(1, 2)
    nkeys = float(Tk)
    got = {}
    o = [torch.matmul(p, vt) for p in P]
    vmax = vt.abs().amax((2, 3), keepdim=True)
    A = [torch.matmul(p, vt.abs()) for p in P]
    w = [1.0] if maps == 1 else [1.0, -lam.double().cpu()[None, :, None, None]]
    out = sum(w[m] * o[m] for m in range(maps))
    eo = sum(abs(w[m]) * ((u + 2 * dS_s[m] + 64 * E) * A[m] + tiny * nkeys * vmax) for m in range(maps)) if maps == 2 else \
        (u + 2 * dS_s[0] + 64 * E) * A[0] + tiny * nkeys * vmax
    rnd = lambda x: u * x.abs() + tiny   # noqa: E731
    tr = lambda x: x.transpose(1, 2)     # noqa: E731
    got["out"] = (tr(out), tr(eo + rnd(out + 0)))
    if maps == 2:
        got["out2"] = (tr(o[1]), tr((u + 2 * dS_s[1] + 64 * E) * A[1] + tiny * nkeys * vmax + rnd(o[1])))
    elow = torch.cat([x.unsqueeze(2) for x in dS_s], 2).flatten(1, 2).squeeze(-1)
    got["lse"] = (lse, elow + 8 * E * torch.where(torch.isfinite(lse), lse.abs(), 0.0))
    if dout is None:
        return got
    do = dout.double().transpose(1, 2)
    W = torch.matmul(do, vt.transpose(2, 3))
    eW = (vt.shape[-1] + 8) * E * torch.matmul(do.abs(), vt.abs().transpose(2, 3))
    # the stored outputs are rounded (and carry eo): their error in D
    eD0 = (do.abs() * (got["out"][1].transpose(1, 2))).sum(-1, keepdim=True) + (do.shape[-1] + 8) * E * (do.abs() * out.abs()).sum(-1, keepdim=True)
    eDs = [eD0]
    if maps == 2:
        eD2 = (do.abs() * got["out2"][1].transpose(1, 2)).sum(-1, keepdim=True) + (do.shape[-1] + 8) * E * (do.abs() * o[1].abs()).sum(-1, keepdim=True)
        eDs = [eD0 + abs(w[1]) * eD2, eD2]
    dS, eS = [], []
    for m in range(maps):
        D = (P[m] * W).sum(-1, keepdim=True)
        x = w[m] * P[m] * (W - D)
        dS.append(x)
        eS.append(2 * dS_s[m] * x.abs() + abs(w[m]) * P[m] * (eW + eDs[m] + 4 * E * (W.abs() + D.abs())))
    Pd = sum(w[m] * P[m] for m in range(maps))
    ePd = sum(abs(w[m]) * 2 * dS_s[m] * P[m] for m in range(maps))
    share = lambda x: x.unflatten(1, (Hkv, G)).sum(2)  # noqa: E731
    dv = share(torch.matmul(Pd.transpose(2, 3), do))
    ev = share(torch.matmul((u * Pd.abs() + ePd + 64 * E * Pd.abs()).transpose(2, 3), do.abs())) + tiny * Tq * G * do.abs().amax()
    got["dv"] = (tr(dv), tr(ev + rnd(dv)))
    dq, dk, eq, ek = [], [], [], []
    for m in range(maps):
        qm, km = q[:, :, m::maps].transpose(1, 2), kk[:, :, m::maps].transpose(1, 2)
        op = eS[m] + (u + 64 * E) * dS[m].abs()
        opt = op + tiny * ok4
        dq.append(torch.matmul(dS[m], km) * scale)
        eq.append(torch.matmul(opt, km.abs()) * scale + rnd(dq[m]))
        dk.append(share(torch.matmul(dS[m].transpose(2, 3), qm)) * scale)
        ek.append(share(torch.matmul(opt.transpose(2, 3), qm.abs())) * scale + rnd(dk[m]))
    weave = lambda xs: torch.stack([tr(x) for x in xs], 3).flatten(2, 3)  # noqa: E731
    got["dq"], got["dk"] = (weave(dq), weave(eq)), (weave(dk), weave(ek))
    if maps == 2:
        x = P[1] * W
        got["dlam"] = (-x.sum((0, 2, 3)), (2 * dS_s[1] * x.abs() + P[1] * eW + 256 * E * x.abs()).sum((0, 2, 3)))
    if table is not None:
        R = buckets.shape[0] // 2
        which = buckets.long()[rel.clamp(-R, R) + R][:, None].expand(B, H, Tq, Tk)
        dt_, et = torch.zeros(table.shape, dtype=torch.float64), torch.zeros(table.shape, dtype=torch.float64)
        for n in range(table.shape[1]):
            hit = which == n
            dt_[:, n] = (dS[0] * hit).sum((0, 2, 3))
            et[:, n] = ((eS[0] + 256 * E * dS[0].abs()) * hit).sum((0, 2, 3))
        got["dtable"] = (dt_, et + rnd(dt_))
    return got


def head_norm(x, w, rope=None, positions=None, eps=1e-6, interleaved=False, alpha=1.0, dy=None):
    """value and bound of y, and with dy of dx and dw; x (B, T, H, d) on the CPU"""
    u, tiny = half_step(x.dtype), (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    xd, wd = x.double(), w.double()
    B, T, H, d = x.shape
    rstd = (xd.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    xh = xd * rstd
    rot = 0 if rope is None else 2 * rope.shape[1]
    ang = None
    if rope is not None:
        pos = torch.arange(T)[None].expand(B, T) if positions is None else positions.long().clamp(0, rope.shape[0] - 1)
        ang = rope.double()[pos].unsqueeze(2)

    def turn(z, sign, mag=False):
        if rope is None:
            return z
        c, s = ang[..., 0], sign * ang[..., 1]
        a, b = (z[..., 0:rot:2], z[..., 1:rot:2]) if interleaved else (z[..., :rot // 2], z[..., rot // 2:rot])
        p, q = (a * c.abs() + b * s.abs(), a * s.abs() + b * c.abs()) if mag else (a * c - b * s, a * s + b * c)
        r = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
        return torch.cat([r, z[..., rot:]], -1)

    y = alpha * turn(xh * wd, 1.0)
    got = {"y": (y, u * y.abs() + tiny + (d / 4 + 16) * E * alpha * turn((xh * wd).abs(), 1.0, True))}
    if dy is None:
        return got
    un = alpha * turn(dy.double(), -1.0)
    um = alpha * turn(dy.double().abs(), 1.0, True)
    uw = un * wd
    mean = (uw * xh).mean(-1, keepdim=True)
    dx = rstd * (uw - xh * mean)
    mag = rstd * (um * wd.abs() + xh.abs() * (um * wd.abs() * xh.abs()).mean(-1, keepdim=True))
    got["dx"] = (dx, u * dx.abs() + tiny + (d / 4 + 24) * E * mag)
    g = (un * xh).sum((0, 1, 2))
    n = B * T * H
    got["dw"] = (g, (min(n, 512 + n // 4096) + d / 4 + 32) * E * (um * xh.abs()).sum((0, 1, 2)))
    return got
