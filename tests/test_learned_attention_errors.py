"""Root-mean-square errors of relative_attention, differential_attention and their gradients: what rounding leaves, and no more
(limits derived in learned_attention_walk.py)."""
import ctypes as C

import pytest
import torch

import learned_attention_walk as W

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
MAPS = pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])


def rnd(*shape, dtype=torch.float32, scale=1.0, seed=0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def inputs(maps, shape, dt, q=1.3, v=1.0, do=1.0, table=1.0, causal=False):
    B, Tq, Tk, H, Hkv, d = shape
    from aniportrait_amd import hipops
    a = dict(q=rnd(B, Tq, maps * H, d, dtype=dt, scale=q, seed=1), k=rnd(B, Tk, maps * Hkv, d, dtype=dt, seed=2),
             v=rnd(B, Tk, Hkv, maps * d, dtype=dt, scale=v, seed=3), do=rnd(B, Tq, H, maps * d, dtype=dt, scale=do, seed=4))
    if maps == 1:
        more = dict(table=rnd(H, 32, dtype=dt, scale=table, seed=5), buckets=hipops.relative_buckets(32, 128, not causal, device="cpu"))
    else:
        more = dict(lam=torch.rand(H, generator=torch.Generator().manual_seed(6)) * 0.6 + 0.2)
    return a, more


def step(maps, a, more, **kw):
    """forward and backward on the GPU -> {name: tensor}"""
    from aniportrait_amd import hipops as ops
    a, more = {n: x.to(DEV) for n, x in a.items()}, [x.to(DEV) for x in more.values()]
    do = a.pop("do")
    fwd, bwd = (ops.relative_attention, ops.relative_attention_backward) if maps == 1 else (ops.differential_attention, ops.differential_attention_backward)
    saved = fwd(*a.values(), *more, for_backward=True, **kw)
    grads = bwd(do, *a.values(), *saved, *more, **kw)
    return dict(zip(("out", "dq", "dk", "dv", "dtable" if maps == 1 else "dlam"), (saved[0], *grads)))


def check(maps, a, more, got=None, exact_d=(), names=("out", "dq", "dk", "dv", "dtable"), causal=False):
    got = got or step(maps, a, more, causal=causal)
    want = W.attention(maps, **a, **more, causal=causal, exact_d=exact_d)
    rel = {n: W.off(got[n], want[n], n) for n in names if n in want}
    assert all(x <= W.LIMIT for x in rel.values()), rel


@MAPS
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_limits_see_small_mistakes(maps, dtype):
    """on the CPU: rounded values pass; values off by 1 %, one head's gradient lost from a shared key head, D left out of one row in
    ten and a bucket without its gradient do not"""
    a, more = inputs(maps, (1, 200, 200, 4, 2, 32), DTYPES[dtype], causal=True)
    want = W.attention(maps, **a, **more, causal=True)
    for n, (ref, _) in want.items():
        good = ref.to(DTYPES[dtype])
        assert W.off(good, want[n]) <= 1.0, n
        if n != "dtable":   # (a few elements, which D's roundings reach: 1 % may be theirs)
            assert W.off(good * 1.01, want[n]) > W.LIMIT, n
    lost = want["dq"][0].clone()
    lost[:, ::10] *= 0.9
    assert W.off(lost, want["dq"]) > W.LIMIT
    half = {n: x.clone() for n, x in a.items()}
    half["do"][:, :, 0] *= 0.97
    other = W.attention(maps, **half, **more, causal=True)
    assert W.off(other["dk"][0], want["dk"]) > W.LIMIT and W.off(other["dv"][0], want["dv"]) > W.LIMIT
    if maps == 1:
        gone = want["dtable"][0].clone()
        gone[0, 7] = 0
        assert W.off(gone, want["dtable"]) > W.LIMIT


SHAPES = [((2, 300, 300, 4, 2, 64), True), ((1, 900, 900, 2, 1, 80), True), ((1, 260, 400, 2, 2, 128), False), ((5, 40, 40, 2, 2, 40), False),
          ((1, 20, 1000, 2, 1, 32), False), ((1, 600, 60, 2, 2, 96), False)]


@pytest.mark.gpu
@MAPS
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape,causal", SHAPES, ids=str)
def test_errors_of_a_training_step(maps, shape, causal, dtype):
    a, more = inputs(maps, shape, DTYPES[dtype], causal=causal)
    check(maps, a, more, causal=causal)


@pytest.mark.gpu
@MAPS
@pytest.mark.parametrize("do,v", [(1e-2, 1.0), (1e-3, 1.0), (1e-4, 1.0), (1e-5, 1.0), (8000.0, 1.0), (1.0, 100.0), (1.0, 1e-3), (1e-3, 300.0), (30.0, 3000.0)])
@pytest.mark.parametrize("shape,causal", [((1, 1000, 1000, 4, 2, 64), True), ((1, 500, 700, 2, 2, 128), False), ((3, 45, 45, 2, 1, 40), False)], ids=str)
def test_fp16_gradients_of_any_size(maps, shape, causal, do, v):
    """small gradients keep their digits, large ones stay finite: dS is rounded as a power of two times itself"""
    a, more = inputs(maps, shape, torch.float16, do=do, v=v, causal=causal)
    check(maps, a, more, causal=causal, names=("dq", "dk", "dv"))


@pytest.mark.gpu
@MAPS
def test_fp16_gradients_of_uneven_size(maps):
    """rows and heads of very different gradients, and values that grow along the keys, in one call"""
    a, more = inputs(maps, (2, 700, 700, 4, 2, 64), torch.float16)
    a["do"] *= torch.logspace(-4, 3, 700)[None, :, None, None].half()
    a["v"] *= torch.logspace(-3, 2.5, 700)[None, :, None, None].half()
    check(maps, a, more, names=("dq", "dk", "dv"))
    a["do"][:, :, 1:] *= 2.0 ** -7
    check(maps, a, more, names=("dq", "dk", "dv"))


PEAKED = [dict(q=8.0), dict(q=16.0), dict(q=4.0, table=8.0)]   # rows whose weight few keys hold


@pytest.mark.gpu
@MAPS
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape,causal", [((1, 1000, 1000, 4, 4, 64), False), ((2, 900, 900, 1, 1, 64), False), ((1, 600, 600, 8, 2, 128), True),
                                          ((20, 150, 150, 2, 2, 40), False)], ids=str)
@pytest.mark.parametrize("sharp", PEAKED, ids=str)
def test_keys_gradients_of_peaked_rows(maps, sharp, shape, causal, dtype):
    """dk takes D from P and W themselves: what the saved outputs' rounding makes of D stays out of it, with whole and split walks"""
    a, more = inputs(maps, shape, DTYPES[dtype], causal=causal, **sharp)
    check(maps, a, more, causal=causal, names=("out", "dk", "dv"), exact_d=("dk",))
    check(maps, a, more, causal=causal, names=("dq", "dtable"))


@pytest.mark.gpu
@MAPS
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape", [(2, 1, 300, 4, 2, 64), (1, 2, 9000, 2, 1, 64), (1, 3, 40000, 1, 1, 40), (300, 3, 40, 2, 2, 32), (2, 200, 200, 2, 2, 64),
                                   (1, 70, 3000, 2, 2, 128)], ids=str)
def test_nan_in_a_query_reaches_its_outputs(maps, shape, dtype):
    """a row whose scores are all NaN is NaN, not one that sees no key; the other rows are as they were"""
    from aniportrait_amd import hipops as ops
    a, more = inputs(maps, shape, DTYPES[dtype], causal=True)
    q, k, v = (a[n].to(DEV) for n in "qkv")
    more = [x.to(DEV) for x in more.values()]
    fwd = ops.relative_attention if maps == 1 else ops.differential_attention
    want = fwd(q, k, v, *more, causal=True, for_backward=True)
    bad = q.clone()
    bad[-1, -1, -1, 3] = float("nan")
    got = fwd(bad, k, v, *more, causal=True, for_backward=True)
    assert got[0][-1, -1, -1].isnan().all() and got[-1][-1, -1, -1].isnan()
    if maps == 2:
        assert got[1][-1, -1, -1].isnan().all()
    rest = torch.ones(got[0].shape[:3], dtype=torch.bool, device=DEV)
    rest[-1, -1, -1] = False
    assert torch.equal(got[0][rest], want[0][rest])


@pytest.mark.gpu
@pytest.mark.parametrize("lam", [0.0, -3.0, 126.0, 129.0, 1000.0, -30000.0])
def test_fp16_differential_attention_of_large_weights(lam):
    """dv is finite where its values are, for any lam; two query heads of a key head with weights of their own"""
    a, more = inputs(2, (1, 400, 400, 4, 2, 64), torch.float16, do=1.0 / (1 + abs(lam)), causal=True)
    more["lam"] = torch.tensor([lam, 0.5, 0.1, lam])
    check(2, a, more, causal=True)


def test_workspace_of_short_sequences_with_a_far_reach():
    """dtable's sums take the diagonals that the sequences have, not those of the reach"""
    from aniportrait_amd import _lib as L
    lib = L.load()
    p = L.AttnParams()
    p.dtype, p.B, p.Tq, p.Tk, p.H, p.Hkv, p.d, p.scale = 1, 1024, 24, 24, 8, 8, 64, 0.125
    for n in ("q", "k", "v", "out", "table", "buckets"):
        setattr(p, n, 256)
    for n in ("q_stride", "k_stride", "v_stride"):
        setattr(p, n, (24 * 512, 512, 64))
    p.n_buckets, p.max_distance = 32, 4096
    tensor = p.B * p.Tq * p.H * p.d * 2
    far = lib.anip_relative_attention_ws_bytes(C.byref(p), 1)
    assert 0 < far <= 2 * tensor
    p.max_distance = 24
    assert lib.anip_relative_attention_ws_bytes(C.byref(p), 1) == far
    p.q_start, p.max_distance = 256, 4096         # (positions of the caller's: any may occur)
    assert lib.anip_relative_attention_ws_bytes(C.byref(p), 1) > 10 * far


@pytest.mark.gpu
@pytest.mark.parametrize("reach", [1, 30, 31, 70, 129, 4096])
@pytest.mark.parametrize("shape,causal", [((40, 20, 20, 2, 1, 32), True), ((3, 70, 30, 2, 2, 64), False), ((2, 30, 300, 2, 2, 128), True),
                                          ((1, 129, 129, 2, 2, 160), False), ((1, 1, 70, 4, 1, 64), False), ((1, 700, 700, 1, 1, 48), False)], ids=str)
def test_table_gradient_of_any_reach(shape, causal, reach):
    """reaches below, at and beyond the distances that the sequences have"""
    a, more = inputs(1, shape, torch.float16, causal=causal)
    r = torch.arange(-reach, reach + 1)
    more["buckets"] = ((r * 7) % 32).int()        # neighbours in different buckets
    check(1, a, more, causal=causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_gradients_at_the_end_of_a_layer(dtype):
    """norm and rotation -> both attentions -> norm of the heads' difference, and back to the projection's rows and all weights: against
    64-bit differentiation of the whole chain.  Each of its up to six roundings in turn (heads, P, output, its norm, the gradients
    between) leaves u / sqrt(3) of a value at most in the mean, errors in D as much again"""
    from aniportrait_amd import hipops as ops
    dt = DTYPES[dtype]
    B, T = 2, 150
    x, g = rnd(B, T, 512, dtype=dt, seed=1), rnd(B, T, 512, dtype=dt, seed=2)
    w = dict(wq=rnd(64, scale=0.2, seed=3) + 1, wk=rnd(64, scale=0.2, seed=4) + 1, wo=rnd(128, scale=0.2, seed=5) + 1, table=rnd(4, 32, dtype=dt, seed=6),
             lam=torch.tensor([0.2, 0.6]))
    rope, buckets = ops.rope_table(T, 64, device="cpu"), ops.relative_buckets(32, 128, False, device="cpu")

    # the framework's operators
    d = {n: t.to(DEV) for n, t in w.items()}
    xd, gd, rd, bd = x.to(DEV), g.to(DEV), rope.to(DEV), buckets.to(DEV)
    q, k, v = xd[..., :256].unflatten(-1, (4, 64)), xd[..., 256:384].unflatten(-1, (2, 64)), xd[..., 384:].unflatten(-1, (2, 64))
    vd = xd[..., 384:].unflatten(-1, (1, 128))
    qn, kn = ops.qk_norm_rope(q, k, d["wq"], d["wk"], rd)
    out, lse = ops.relative_attention(qn, kn, v, d["table"], bd, causal=True, for_backward=True)
    od, od2, lsed = ops.differential_attention(qn, kn, vd, d["lam"], causal=True, for_backward=True)
    on, _ = ops.qk_norm_rope(od, None, d["wo"], None)
    g1, g2 = gd[..., :256].unflatten(-1, (4, 64)), gd[..., 256:].unflatten(-1, (2, 128))
    god, _, dwo, _ = ops.qk_norm_rope_backward(g2, None, od, None, d["wo"], None)
    r = ops.relative_attention_backward(g1, qn, kn, v, out, lse, d["table"], bd, causal=True)
    s = ops.differential_attention_backward(god, qn, kn, vd, od, od2, lsed, d["lam"], causal=True)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(r[0] + s[0], r[1] + s[1], q, k, d["wq"], d["wk"], rd)
    dx = torch.cat([dq.flatten(2), dk.flatten(2), r[2].flatten(2) + s[2].flatten(2)], -1)
    got = dict(x=dx, wq=dwq, wk=dwk, wo=dwo, table=r[3], lam=s[3], y=torch.cat([out.flatten(2), on.flatten(2)], -1))

    # the definition
    p = {n: t.double().requires_grad_() for n, t in dict(w, x=x).items()}
    turn = torch.view_as_complex(rope.double())[:, None]

    def norm(h, weight):
        return h * (h.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * weight

    def rotate(h):
        z = torch.complex(*h.chunk(2, -1)) * turn
        return torch.cat([z.real, z.imag], -1)
    q, k = p["x"][..., :256].unflatten(-1, (4, 64)), p["x"][..., 256:384].unflatten(-1, (2, 64))
    v, vd = p["x"][..., 384:].unflatten(-1, (2, 64)), p["x"][..., 384:].unflatten(-1, (1, 128))
    qn, kn = rotate(norm(q, p["wq"])), rotate(norm(k, p["wk"]))
    rel = torch.arange(T)[None] - torch.arange(T)[:, None]

    def maps(qh, kh, bias):
        z = torch.einsum("bihc,bjhc->bhij", qh, kh) / 8 + bias
        return z.masked_fill(rel > 0, -float("inf")).softmax(-1)
    P = maps(qn, kn.repeat_interleave(2, 2), p["table"][:, buckets.long()[rel.clamp(-128, 128) + 128]])
    y1 = torch.einsum("bhij,bjhc->bihc", P, v.repeat_interleave(2, 2))
    A = [maps(qn[:, :, m::2], kn[:, :, m::2].expand(-1, -1, 2, -1), 0.0) for m in (0, 1)]
    o2 = torch.einsum("bhij,bjhc->bihc", A[1], vd.expand(-1, -1, 2, -1))
    o = torch.einsum("bhij,bjhc->bihc", A[0], vd.expand(-1, -1, 2, -1)) - p["lam"][:, None] * o2
    y2 = norm(o, p["wo"])
    y = torch.cat([y1.flatten(2), y2.flatten(2)], -1)
    *grads, go = torch.autograd.grad(y, [*p.values(), o], g.double())
    want = dict(zip(p, grads), y=y.detach())
    limit = 2 * (6 / 3) ** 0.5 * torch.finfo(dt).eps / 2
    # dlam = -sum go o2 over 38400 terms a head, whose roundings add up as the root of their squares while they cancel themselves: the
    # norm's gradient go is at right angles to o in every row, and o2 lies mostly along o
    size = {n: ref.norm() for n, ref in want.items()}
    size["lam"] = (go * o2).norm()
    assert size["lam"] > 2 * want["lam"].norm()
    rel_err = {n: ((got[n].cpu().double() - ref).norm() / size[n]).item() for n, ref in want.items()}
    for part, sl in (("dq", slice(0, 256)), ("dk", slice(256, 384)), ("dv", slice(384, 512))):
        rel_err[part] = ((got["x"].cpu().double() - want["x"])[..., sl].norm() / want["x"][..., sl].norm()).item()
    assert all(e <= limit for e in rel_err.values()), (limit, rel_err)
    # a hand-over that drops one attention's gradient is seen: it is ten times the limit at least
    assert (r[0].norm() / dq.norm()).item() > 10 * limit and (s[0].norm() / dq.norm()).item() > 10 * limit


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 200, 230, 2, 2, 64), (2, 3, 230, 4, 2, 40), (1, 900, 900, 1, 1, 64)], ids=str)
def test_lowest_bias_of_bf16_hides(shape):
    """bf16's lowest value times log2 e is beyond 32 bits: it hides its pairs as -inf does, and rows without others are zeros"""
    a, more = inputs(1, shape, torch.bfloat16)
    res = []
    for low in (torch.finfo(torch.bfloat16).min, -float("inf")):
        table = more["table"].clone()
        table[:, ::3] = low
        table[0, :] = low
        res.append(step(1, a, dict(more, table=table), q_start=torch.full((shape[0],), 5, dtype=torch.int32, device=DEV)))
    for n in res[0]:
        assert torch.equal(res[0][n], res[1][n]) and res[0][n].isfinite().all(), n
    assert res[0]["out"][:, :, 0].abs().max() == 0 and res[0]["dq"][:, :, 0].abs().max() == 0 and res[0]["dtable"][0].abs().max() == 0


@pytest.mark.gpu
@MAPS
@pytest.mark.parametrize("odd", ["large", "nan", "inf", "nan query"])
def test_fp16_rows_beside_an_odd_one(maps, odd):
    """a query whose gradient passes fp16's range, or is none, leaves the other waves' rows of its workgroup their precision; NaN also its own wave's"""
    a, more = inputs(maps, (1, 400, 400, 2, 2, 64), torch.float16)
    if odd == "large":       # its dS reaches 1e6
        a["do"][0, 5] *= 2000
        a["v"][0, 7] *= 300
        a["q"][0, 5] = a["k"][0, 7] * 2
    want = W.attention(maps, **a, **more)
    bad = {n: x.clone() for n, x in a.items()}
    if odd in ("nan", "inf"):
        bad["do"][0, 5, :, 3] = float(odd)
    elif odd == "nan query":
        bad["q"][0, 5, :, 3] = float("nan")
    got = step(maps, bad, more)
    rest = torch.arange(400) >= 32 if odd == "large" else torch.arange(400) != 5
    for lo, hi in ((0, 128), (128, 400)):
        part = rest & (torch.arange(400) >= lo) & (torch.arange(400) < hi)
        e = W.off(got["dq"][:, part], tuple(x[:, part] for x in want["dq"]))
        assert e <= W.LIMIT, (lo, e)
    if odd != "large":
        assert got["dq"][0, 5].isnan().all()
        assert got["out"][0, 6:].isfinite().all()
