"""Root-mean-square errors that rounding leaves in the outputs of relative_attention and differential_attention, for limits that a
wrong factor, a lost term or a lost digit cannot pass (learned_attention_oracle's bounds add every rounding's worst case).

Roundings are independent and uniform, within half a step u of the value, so u^2 / 3 of its square at most in the mean.  With v() the
mean square error of a value:
  out   u^2/3 (out^2 + sum (w P V)^2)                    its own rounding, and P's as operand of the product
  D     sum dO^2 v(stored outputs)                        where it is taken from those
  dq    u^2/3 (dq^2 + scale^2 sum dS^2 K^2)  + scale^2 (w sum P K)^2 v(D)
  dk    u^2/3 (dk^2 + scale^2 sum dS^2 Q^2)  + scale^2 sum (w P Q)^2 v(D)
  dv    u^2/3 (dv^2 + sum P^2 dO^2)
  dtable  u^2/3 dtable^2 + sum over rows (sum of P over the bucket)^2 v(D), beyond the bias's reach without the last
and (2^-25)^2 / 3 for each fp16 output that may lie below 2^-14.  32-bit sums are 2^-16 of that and not counted."""
import math

import torch


def attention(maps, q, k, v, do, causal=False, table=None, buckets=None, lam=None, exact_d=(), lens=None):
    """{name: (value in 64 bits, mean square error)}; CPU tensors in the framework's layouts; exact_d: the outputs whose D is exact"""
    dt = q.dtype
    c = (torch.finfo(dt).eps / 2) ** 2 / 3
    tiny = (2.0 ** -25) ** 2 / 3 if dt == torch.float16 else 0.0
    B, Tq, _, d = q.shape
    Tk, Hkv = v.shape[1:3]
    H = q.shape[2] // maps
    G, scale = H // Hkv, d ** -0.5
    rel = torch.arange(Tk)[None] - (torch.arange(Tq)[:, None] + Tk - Tq)
    hide = ((rel > 0) if causal else torch.zeros_like(rel, dtype=torch.bool)).expand(B, 1, Tq, Tk)
    if lens is not None:
        hide = hide | (torch.arange(Tk)[None, :] >= torch.tensor(lens)[:, None])[:, None, None]
    q, k, v, do = (x.double().transpose(1, 2) for x in (q, k, v, do))
    share = lambda x: x.unflatten(1, (Hkv, G)).sum(2)   # noqa: E731
    V = v.repeat_interleave(G, 1)
    P, W = [], do @ V.transpose(2, 3)
    w = [1.0] if maps == 1 else [1.0, -lam.double()[None, :, None, None]]
    K = [k[:, m::maps].repeat_interleave(G, 1) for m in range(maps)]
    Q = [q[:, m::maps] for m in range(maps)]
    for m in range(maps):
        s = Q[m] @ K[m].transpose(2, 3) * scale
        if table is not None:
            R = buckets.numel() // 2
            which = buckets.long()[rel.clamp(-R, R) + R]
            s = s + table.double()[:, which]
        s = s.masked_fill(hide, -math.inf)
        P.append(torch.nan_to_num((s - s.amax(-1, keepdim=True)).softmax(-1), 0.0))
    o = [p @ V for p in P]
    out = sum(a * x for a, x in zip(w, o))
    vo = [c * (p ** 2) @ (V ** 2) for p in P]
    got = {"out": (out, c * out ** 2 + tiny + sum(a ** 2 * x for a, x in zip(w, vo)))}
    saved = [got["out"][1]] if maps == 1 else [got["out"][1] + w[1] ** 2 * (c * o[1] ** 2 + vo[1]), c * o[1] ** 2 + vo[1]]
    dq, dk = [], []
    for m in range(maps):
        vD = (do ** 2 * saved[m]).sum(-1, keepdim=True)
        dS = w[m] * P[m] * (W - (P[m] * W).sum(-1, keepdim=True))
        x = dS @ K[m] * scale
        e = c * (x ** 2 + scale ** 2 * (dS ** 2) @ (K[m] ** 2)) + tiny
        dq.append((x, e + (0.0 if "dq" in exact_d else scale ** 2 * (w[m] * P[m] @ K[m]) ** 2 * vD)))
        x = share(dS.transpose(2, 3) @ Q[m] * scale)
        e = c * (x ** 2 + scale ** 2 * share((dS ** 2).transpose(2, 3) @ (Q[m] ** 2))) + tiny
        dk.append((x, e + (0.0 if "dk" in exact_d else scale ** 2 * share(((w[m] * P[m]) ** 2 * vD).transpose(2, 3) @ (Q[m] ** 2)))))
        if m == 0 and table is not None:
            near = rel.abs() < R
            t, et = torch.zeros_like(table, dtype=torch.float64), torch.zeros_like(table, dtype=torch.float64)
            for n in range(table.shape[1]):
                hit = which == n
                t[:, n] = (dS * hit).sum((0, 2, 3))
                et[:, n] = ((P[0] * (hit & near)).sum(-1) ** 2 * vD.squeeze(-1)).sum((0, 2))
            got["dtable"] = (t, c * t ** 2 + tiny + et)
    Pd = sum(a * p for a, p in zip(w, P))
    dv = share(Pd.transpose(2, 3) @ do)
    got["dv"] = (dv, c * (dv ** 2 + share((Pd ** 2).transpose(2, 3) @ (do ** 2))) + tiny)
    for n, x in (("dq", dq), ("dk", dk)):
        got[n] = tuple(torch.stack([y[i] for y in x], 2).flatten(1, 2) for i in (0, 1))
    return {n: (a.transpose(1, 2), b.transpose(1, 2)) if n != "dtable" else (a, b) for n, (a, b) in got.items()}


def off(got, want, name=None):
    """the root-mean-square error over what rounding accounts for"""
    ref, e = want
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, name
    fit = ref.abs() < torch.finfo(torch.float16).max   # (what fp16 cannot hold is infinite on either side)
    return ((got - ref)[fit].pow(2).mean() / e[fit].mean()).sqrt().item()


LIMIT = 1.5   # of off(): u^2 / 3 is 1.8 times a rounding's mean square over a decade of values; the rest is chance in few elements
