"""qk_norm_rope, relative_attention, differential_attention and their gradients against 64-bit definitions, element by element
within bounds derived in learned_attention_oracle.py; their refusals; and the ways they are called."""
import ctypes as C
import math

import pytest
import torch

import learned_attention_oracle as O

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _ops():
    from aniportrait_amd import hipops
    return hipops


def rnd(*shape, dtype=torch.float32, scale=1.0, shift=0.0, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + sum((i + 1) * s for i, s in enumerate(shape)))
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype)


def within(got, want, name):
    ref, tol = want
    got = got.detach().cpu()
    assert tuple(got.shape) == tuple(ref.shape), f"{name}: shape {tuple(got.shape)} for {tuple(ref.shape)}"
    got = got.double()
    fin = torch.isfinite(ref)
    assert torch.equal(fin, torch.isfinite(got)), f"{name}: not finite at {(fin != torch.isfinite(got)).nonzero()[:3].tolist()}"
    assert torch.equal(got[~fin], ref[~fin]), f"{name}: other infinities"
    err = (got - ref).abs()[fin]
    over = err - tol[fin] - 1e-30
    assert not (over > 0).any(), (f"{name}: {int((over > 0).sum())} of {err.numel()} out of bounds, worst {err.max().item():.3e} "
                                  f"of rms {ref[fin].pow(2).mean().sqrt().item():.3e}, worst ratio {(err / (tol[fin] + 1e-30)).max().item():.2f}, "
                                  f"at {((got - ref).abs() - tol > 0).nonzero()[:3].tolist()}")


# ---------------------------------------------------------------------------------------------------------------
# refusals that need no GPU: the library's own checks, ahead of any launch
# ---------------------------------------------------------------------------------------------------------------
def _attn_params(maps, **kw):
    from aniportrait_amd import _lib as L
    p = L.AttnParams()
    p.dtype, p.B, p.Tq, p.Tk, p.H, p.Hkv, p.d, p.causal, p.scale = 0, 2, 64, 64, 4, 2, 64, 0, 0.125
    for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv", "lse"):
        setattr(p, n, 256)
    for n in ("q_stride", "k_stride", "v_stride", "dout_stride"):
        setattr(p, n, (64 * 256, 256, 64))
    if maps == 1:
        p.table, p.buckets, p.n_buckets, p.max_distance, p.dtable = 256, 256, 32, 128, 256
    else:
        p.lam, p.out2, p.dlam = 256, 256, 256
    for n, v in kw.items():
        setattr(p, n, v)
    return p


BAD = [dict(dtype=2), dict(B=0), dict(Tq=0), dict(Tk=0), dict(H=3), dict(H=0), dict(Hkv=0), dict(d=0), dict(d=12), dict(d=168), dict(scale=0.0),
       dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=0), dict(k=264), dict(v=0), dict(out=0),
       dict(q_stride=(64 * 256, 252, 64)), dict(k_stride=(64 * 256, 1 << 24, 64)), dict(v_stride=(64 * 256, -256, 64)),
       dict(Tq=(1 << 28) + 1), dict(H=1 << 21, Hkv=1 << 21), dict(B=1 << 30), dict(out2=8)]


@pytest.mark.parametrize("maps", [1, 2])
@pytest.mark.parametrize("bad", BAD + [dict(table=0, lam=0), dict(n_buckets=0, lam=0), dict(max_distance=4097, lam=0)],
                         ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_attention_refuses(maps, bad):
    lib = _ops().L.load()
    name = "anip_relative_attention" if maps == 1 else "anip_differential_attention"
    p = _attn_params(maps, **bad)
    assert getattr(lib, name)(C.byref(p), None) == -1
    assert name.encode() in lib.anip_last_error()
    assert getattr(lib, name + "_backward")(C.byref(p), None) == -1
    assert getattr(lib, name + "_ws_bytes")(C.byref(p), 0) == -1
    assert getattr(lib, name)(None, None) == -1


@pytest.mark.parametrize("maps,bad", [(1, dict(dtable=0)), (2, dict(dlam=0)), (2, dict(out2=0)), (1, dict(lse=0)), (2, dict(dq=0)), (1, dict(dk=0)),
                                      (1, dict(dv=0)), (2, dict(dq=264)), (1, dict(dk=8)), (2, dict(dout=0)), (1, dict(dout_stride=(8, 4, 8))), (1, {}), (2, dict(workspace=256, workspace_bytes=64))])
def test_attention_backward_refuses(maps, bad):
    """missing outputs, and a workspace that is missing or too small"""
    lib = _ops().L.load()
    name = "anip_relative_attention" if maps == 1 else "anip_differential_attention"
    p = _attn_params(maps, **bad)
    assert getattr(lib, name + "_backward")(C.byref(p), None) == -1
    assert (name + "_backward").encode() in lib.anip_last_error()


def test_split_forward_wants_its_workspace():
    lib = _ops().L.load()
    p = _attn_params(1, B=1, Tq=1, Tk=8192, H=4, Hkv=4)
    need = lib.anip_relative_attention_ws_bytes(C.byref(p), 0)
    assert need > 0 and need % (4 * 65 * 4) == 0
    assert lib.anip_relative_attention(C.byref(p), None) == -1 and b"workspace" in lib.anip_last_error()
    assert lib.anip_relative_attention_ws_bytes(C.byref(_attn_params(1, B=64, Tq=512, Tk=512)), 0) == 0


@pytest.mark.parametrize("maps", [1, 2])
def test_stride_of_a_lone_token_is_not_looked_at(maps):
    lib = _ops().L.load()
    f = lib.anip_relative_attention_ws_bytes if maps == 1 else lib.anip_differential_attention_ws_bytes
    far = (64 * 256, 1 << 25, 64)
    assert f(C.byref(_attn_params(maps, Tq=1, q_stride=far)), 0) >= 0
    assert f(C.byref(_attn_params(maps, Tk=1, k_stride=far, v_stride=far)), 0) >= 0
    assert f(C.byref(_attn_params(maps, Tk=1, q_stride=far)), 0) == -1


def _norm_params(**kw):
    from aniportrait_amd import _lib as L
    p = L.QkNormParams()
    p.dtype, p.B, p.T, p.Hq, p.Hkv, p.d, p.rot, p.eps, p.q_alpha = 0, 2, 8, 4, 2, 64, 64, 1e-6, 1.0
    for n in ("q", "k", "q_out", "k_out", "q_weight", "k_weight", "rope", "dq_out", "dk_out", "dq_weight", "dk_weight", "ws"):
        setattr(p, n, 256)
    p.rope_rows, p.ws_floats = 8, 1 << 20
    for n in ("q", "k", "q_out", "k_out", "dq_out", "dk_out"):
        setattr(p, n + "_stride", (8 * 256, 256, 64))
    for n, v in kw.items():
        setattr(p, n, v)
    return p


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(B=0), dict(T=0), dict(Hq=0), dict(Hkv=-1), dict(d=4), dict(d=264), dict(rot=4), dict(rot=72), dict(rope=0),
                                 dict(rope=264), dict(rope_rows=0), dict(rope_rows=7), dict(q=0), dict(k=8), dict(q_weight=0), dict(k_weight=0),
                                 dict(q_out=0), dict(k_out=264), dict(q_stride=(8, 4, 8)), dict(k_out_stride=(8, 8, 4)), dict(T=1 << 30)],
                         ids=lambda b: "-".join(f"{k}={v}" for k, v in b.items()))
def test_qk_norm_rope_refuses(bad):
    lib = _ops().L.load()
    p = _norm_params(**bad)
    assert lib.anip_qk_norm_rope(C.byref(p), None) == -1 and b"anip_qk_norm_rope" in lib.anip_last_error()
    assert lib.anip_qk_norm_rope_backward(C.byref(p), None) == -1
    assert lib.anip_qk_norm_rope(None, None) == -1


@pytest.mark.parametrize("bad", [dict(ws=0), dict(ws_floats=1), dict(dq_weight=0), dict(dk_weight=0), dict(dq_out=0), dict(dk_out=8)])
def test_qk_norm_rope_backward_refuses(bad):
    lib = _ops().L.load()
    assert lib.anip_qk_norm_rope_backward(C.byref(_norm_params(**bad)), None) == -1


def test_wrappers_refuse_cpu_tensors():
    ops = _ops()
    x = torch.zeros((1, 8, 2, 64), dtype=torch.float16)
    with pytest.raises(ops.L.HipLibraryError):
        ops.qk_norm_rope(x, x, torch.ones(64), torch.ones(64))
    with pytest.raises(ops.L.HipLibraryError):
        ops.relative_attention(x, x, x, torch.zeros((2, 32), dtype=torch.float16), ops.relative_buckets(32, 128, device="cpu"))
    with pytest.raises(ops.L.HipLibraryError):
        ops.differential_attention(x, x, torch.zeros((1, 8, 1, 128), dtype=torch.float16), torch.zeros(1))


def test_struct_mirrors_match_the_header():
    import os
    import re
    from aniportrait_amd import _lib as L
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "aniportrait_hip.h")).read()
    for name, mirror in (("anip_qk_norm_params", L.QkNormParams), ("anip_attn_params", L.AttnParams)):
        body = src[src.index("typedef struct " + name + " {"):src.index("} " + name + ";")]
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S).split("{", 1)[1]
        fields = []
        for stmt in body.split(";"):
            for part in stmt.split(","):
                ids = re.findall(r"[A-Za-z_][A-Za-z0-9_]*", re.sub(r"\[\d+\]", "", part))
                if ids:
                    fields.append(ids[-1])
        assert fields == [f[0] for f in mirror._fields_], name


@pytest.mark.parametrize("nb,md,bi", [(32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (64, 4096, True), (7, 11, False), (320, 800, True)])
def test_relative_buckets(nb, md, bi):
    """monotone away from zero, exact near it, every bucket's border where the definition puts it"""
    got = _ops().relative_buckets(nb, md, bi, device="cpu").tolist()
    assert len(got) == 2 * md + 1
    side = nb // 2 if bi else nb
    exact, s = side // 2, side - side // 2
    for r in range(-md, md + 1):
        n = abs(r) if bi else max(-r, 0)
        if n < exact:
            want = n
        else:
            want = exact + max(j for j in range(s) if n ** s * exact ** j >= md ** j * exact ** s) if n < md else side - 1
        assert got[r + md] == want + (side if bi and r > 0 else 0), r
    for bad in ((3, 128, True), (2, 128, True), (1, 8, False), (32, 8, True), (5, 64, True)):
        with pytest.raises(ValueError):
            _ops().relative_buckets(*bad, device="cpu")


# ---------------------------------------------------------------------------------------------------------------
# qk_norm_rope
# ---------------------------------------------------------------------------------------------------------------
NORMS = [  # B, T, Hq, Hkv, d, rot, interleaved, far
    (1, 1, 1, 1, 8, 8, False, False), (2, 1, 32, 8, 128, 128, False, True), (2, 77, 4, 2, 40, 40, False, False),
    (1, 130, 3, 1, 80, 40, True, True), (3, 50, 5, 5, 64, 0, False, False), (1, 300, 2, 1, 160, 160, True, False),
    (2, 33, 2, 2, 256, 64, False, True), (1, 1500, 8, 8, 32, 32, True, False), (2, 9, 7, 0, 96, 96, False, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,T,Hq,Hkv,d,rot,inter,far", NORMS)
def test_qk_norm_rope(B, T, Hq, Hkv, d, rot, inter, far, dtype):
    ops, dt = _ops(), DTYPES[dtype]
    qkv = rnd(B, T, (Hq + 2 * Hkv) * d, dtype=dt, scale=2.0, seed=1)
    qkv[0, 0, :d] = 0.0                                  # a head of zeros
    q, k = qkv[..., :Hq * d].unflatten(-1, (Hq, d)), (qkv[..., Hq * d:(Hq + Hkv) * d].unflatten(-1, (Hkv, d)) if Hkv else None)
    wq, wk = rnd(d, scale=0.3, shift=1.0, seed=2), (rnd(d, scale=0.3, shift=1.0, seed=3) if Hkv else None)
    n = 70000 if far else T
    rope = ops.rope_table(n, rot, device="cpu") if rot else None
    pos = torch.randint(0, n, (B, T), generator=torch.Generator().manual_seed(5), dtype=torch.int32) if far and rot else None
    if pos is not None and T > 2:
        pos[0, 1], pos[0, 2] = -5, n + 7                 # outside the table: its ends
    kw = dict(eps=1e-5, interleaved=inter, q_alpha=0.37)
    g = lambda t: None if t is None else t.to(DEV)       # noqa: E731
    qkv_d = qkv.to(DEV)
    qd, kd = qkv_d[..., :Hq * d].unflatten(-1, (Hq, d)), (qkv_d[..., Hq * d:(Hq + Hkv) * d].unflatten(-1, (Hkv, d)) if Hkv else None)
    qo, ko = ops.qk_norm_rope(qd, kd, g(wq), g(wk), g(rope), g(pos), **kw)
    gq, gk = rnd(B, T, Hq, d, dtype=dt, seed=7), (rnd(B, T, Hkv, d, dtype=dt, seed=8) if Hkv else None)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(g(gq), g(gk), qd, kd, g(wq), g(wk), g(rope), g(pos), **kw)
    wantq = O.head_norm(q, wq, rope, pos, 1e-5, inter, 0.37, gq)
    for name, x, y in (("q", qo, "y"), ("dq", dq, "dx"), ("dwq", dwq, "dw")):
        within(x, wantq[y], name)
    if Hkv:
        wantk = O.head_norm(k, wk, rope, pos, 1e-5, inter, 1.0, gk)
        for name, x, y in (("k", ko, "y"), ("dk", dk, "dx"), ("dwk", dwk, "dw")):
            within(x, wantk[y], name)
    else:
        assert ko is None and dk is None and dwk is None
    # in place, into the fused projection itself: the same bits, the value heads untouched
    before = qkv_d.clone()
    ops.qk_norm_rope(qd, kd, g(wq), g(wk), g(rope), g(pos), q_out=qd, k_out=kd, **kw)
    assert torch.equal(qd, qo) and (ko is None or torch.equal(kd, ko))
    assert torch.equal(qkv_d[..., (Hq + Hkv) * d:], before[..., (Hq + Hkv) * d:])


@pytest.mark.gpu
def test_qk_norm_rope_into_a_cache():
    """new keys written into their place of a longer cache: the rest of it stays"""
    ops = _ops()
    q, k, w = rnd(2, 3, 4, 64, dtype=torch.bfloat16, seed=1).to(DEV), rnd(2, 3, 2, 64, dtype=torch.bfloat16, seed=2).to(DEV), torch.ones(64, device=DEV)
    cache = rnd(2, 50, 2, 64, dtype=torch.bfloat16, seed=3).to(DEV)
    before = cache.clone()
    _, want = ops.qk_norm_rope(q, k, w, w)
    _, got = ops.qk_norm_rope(q, k, w, w, k_out=cache[:, 20:23])
    assert got.data_ptr() == cache[:, 20:23].data_ptr() and torch.equal(cache[:, 20:23], want)
    assert torch.equal(cache[:, :20], before[:, :20]) and torch.equal(cache[:, 23:], before[:, 23:])


@pytest.mark.gpu
def test_qk_norm_rope_without_eps():
    """eps = 0 is a legal value: heads that do not exist in a group add nothing to the weights' gradient"""
    ops = _ops()
    q, k = rnd(1, 1000, 9, 64, dtype=torch.float16, seed=1), rnd(1, 1000, 3, 64, dtype=torch.float16, seed=2)
    w = rnd(64, shift=1.0, scale=0.2, seed=3)
    gq, gk = rnd(1, 1000, 9, 64, dtype=torch.float16, seed=4), rnd(1, 1000, 3, 64, dtype=torch.float16, seed=5)
    r = ops.qk_norm_rope_backward(gq.to(DEV), gk.to(DEV), q.to(DEV), k.to(DEV), w.to(DEV), w.to(DEV), eps=0.0)
    for x, g, dx, dw in ((q, gq, r[0], r[2]), (k, gk, r[1], r[3])):
        want = O.head_norm(x, w, eps=0.0, dy=g)
        within(dx, want["dx"], "dx")
        within(dw, want["dw"], "dw")


@pytest.mark.gpu
def test_qk_norm_rope_gradient_against_differences():
    """the backward's dx along a direction against central differences of the 64-bit forward"""
    ops = _ops()
    x, w, rope = rnd(1, 5, 2, 64, dtype=torch.float16, seed=1), rnd(64, shift=1.0, scale=0.2, seed=2), ops.rope_table(5, 32, device="cpu")
    gy, step = rnd(1, 5, 2, 64, dtype=torch.float16, seed=3), rnd(1, 5, 2, 64, seed=4).double()
    dx, _, dw, _ = ops.qk_norm_rope_backward(gy.to(DEV), None, x.to(DEV), None, w.to(DEV), None, rope.to(DEV))

    def f(xx, ww):
        big = O.head_norm(xx, ww, rope)["y"][0]
        return (big * gy.double()).sum().item()
    h = 1e-5
    x64 = x.double()
    num = (f(x64 + h * step, w) - f(x64 - h * step, w)) / (2 * h)
    ana = (dx.cpu().double() * step).sum().item()
    # dx is rounded to fp16: |error| <= 2^-11 sum |dx||step|; the differences' own error is h^2 and 1e-16 / h
    assert abs(num - ana) <= 2.0 ** -11 * (dx.cpu().double().abs() * step.abs()).sum().item() + 1e-6 * (1 + abs(num))


# ---------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------
def _inputs(maps, B, Tq, Tk, H, Hkv, d, dt, lens, fused=False, seed=1):
    q = rnd(B, Tq, maps * H, d, dtype=dt, scale=1.3, seed=seed)
    k = rnd(B, Tk, maps * Hkv, d, dtype=dt, seed=seed + 1)
    v = rnd(B, Tk, Hkv, maps * d, dtype=dt, seed=seed + 2)
    do = rnd(B, Tq, H, maps * d, dtype=dt, seed=seed + 3)
    lens_t = None if lens is None else torch.tensor(lens, dtype=torch.int32)
    if lens is not None:
        for b, n in enumerate(lens):   # nothing behind a sequence's end may be used
            n = min(max(n, 0), Tk)
            k[b, n:], v[b, n:] = float("nan"), float("inf")
    return q, k, v, do, lens_t


def _strided(t, dev=DEV):
    """the same values with another layout: (head, batch, token, channel) in memory, 8 channels of padding"""
    B, T, H, d = t.shape
    big = torch.full((H, B, T, d + 8), float("nan"), dtype=t.dtype, device=dev)
    big[..., :d] = t.to(dev).permute(2, 0, 1, 3)
    return big[..., :d].permute(1, 2, 0, 3)


def _check(maps, shape, dtype, causal=False, lens=None, start=None, scale=None, extra=None, strided=False, train=True):
    ops, dt = _ops(), DTYPES[dtype]
    B, Tq, Tk, H, Hkv, d = shape
    q, k, v, do, lens_t = _inputs(maps, B, Tq, Tk, H, Hkv, d, dt, lens)
    start_t = None if start is None else torch.tensor(start, dtype=torch.int32)
    kw = dict(causal=causal, scale=scale, kv_lens=None if lens_t is None else lens_t.to(DEV), q_start=None if start_t is None else start_t.to(DEV))
    put = _strided if strided else (lambda t: t.to(DEV))
    qd, kd, vd, dd = put(q), put(k), put(v), put(do)
    if maps == 1:
        table, buckets = extra or (rnd(H, 32, dtype=dt, seed=9), ops.relative_buckets(32, 128, not causal, device="cpu"))
        lam = None
        call = (table.to(DEV), buckets.to(DEV))
        out, lse = ops.relative_attention(qd, kd, vd, *call, for_backward=True, **kw)
        again = ops.relative_attention(qd, kd, vd, *call, **kw)
        got = dict(out=out, lse=lse)
        if train:
            got.update(zip(("dq", "dk", "dv", "dtable"), ops.relative_attention_backward(dd, qd, kd, vd, out, lse, *call, **kw)))
    else:
        table = buckets = None
        lam = extra if extra is not None else torch.rand(H, generator=torch.Generator().manual_seed(3)) * 0.8
        ld = lam.to(DEV)
        out, out2, lse = ops.differential_attention(qd, kd, vd, ld, for_backward=True, **kw)
        again = ops.differential_attention(qd, kd, vd, ld, **kw)
        got = dict(out=out, out2=out2, lse=lse)
        if train:
            got.update(zip(("dq", "dk", "dv", "dlam"), ops.differential_attention_backward(dd, qd, kd, vd, out, out2, lse, ld, **kw)))
    assert torch.equal(again, out)
    want = O.attention(maps, q, k, v, causal, scale, lens_t, start_t, table, buckets, lam, do if train else None)
    for name, x in got.items():
        within(x, want[name], name)
    return got


SHAPES = [  # (B, Tq, Tk, H, Hkv, d), causal, lens, start
    ((1, 1, 1, 1, 1, 8), False, None, None),
    ((2, 1, 77, 4, 2, 64), True, None, None),
    ((2, 33, 33, 2, 2, 40), False, None, None),
    ((1, 128, 128, 2, 1, 64), True, None, None),
    ((1, 129, 200, 3, 3, 80), False, None, None),
    ((1, 300, 300, 4, 2, 128), True, None, None),
    ((3, 50, 170, 2, 2, 32), False, [0, 1, 170], None),
    ((4, 70, 70, 2, 1, 48), True, [70, 0, 33, 64], None),
    ((2, 5, 300, 6, 2, 16), True, [300, 41], [295, 36]),
    ((2, 130, 90, 2, 2, 24), True, None, [-70, 20]),        # queries ahead of the first key: rows without keys
    ((1, 64, 64, 2, 2, 64), True, None, [1000000]),         # far positions
    ((2, 65, 31, 1, 1, 72), False, [-3, 99], [5, -5]),      # lengths outside [0, Tk]
    ((1, 40, 2100, 2, 2, 64), True, None, None),            # keys split over workgroups
    ((2, 1, 3001, 8, 2, 128), True, [3001, 1700], [3000, 1699]),
    ((1, 257, 257, 1, 1, 120), False, None, None),
    ((1, 900, 900, 4, 1, 64), True, None, None),            # both walks of the backward split
    ((1, 1000, 40, 2, 2, 128), False, [37], None)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shape,causal,lens,start", SHAPES, ids=lambda x: str(x))
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention(maps, shape, causal, lens, start, dtype):
    _check(maps, shape, dtype, causal, lens, start)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,causal", [((1, 100, 100, 2, 2, 160), True), ((2, 1, 500, 5, 1, 160), False), ((1, 200, 150, 1, 1, 144), False)])
def test_relative_attention_widest_heads(shape, causal):
    _check(1, shape, "fp16", causal, start=[3] if shape[0] == 1 else None)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention_of_many_short_sequences(maps):
    """a wave per problem: the motion modules' shape, an odd number of problems"""
    _check(maps, (701, 5, 7, 3, 3, 40), "fp16", lens=[i % 8 for i in range(701)])


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
@pytest.mark.parametrize("shape", [(2, 70, 150, 2, 1, 64), (2, 3, 150, 4, 2, 40)])
def test_attention_of_strided_tensors(maps, shape):
    _check(maps, shape, "bf16", True, strided=True)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_lone_tokens_of_far_strides(maps):
    """one query or one key cut from a token-major tensor of very long rows"""
    ops, dt = _ops(), torch.float16
    far = lambda t: t.as_strided(t.shape, (t.stride(0), 1 << 25, t.stride(2), 1)) if t.shape[1] == 1 else t   # noqa: E731
    for Tq, Tk in ((1, 50), (40, 1), (1, 1)):
        q, k, v, do, _ = (x if x is None else x.to(DEV) for x in _inputs(maps, 1, Tq, Tk, 2, 2, 64, dt, None))
        if maps == 1:
            more = (rnd(2, 32, dtype=dt, seed=9).to(DEV), ops.relative_buckets(32, 128, device=DEV))
            fwd, bwd = ops.relative_attention, ops.relative_attention_backward
        else:
            more, fwd, bwd = (torch.tensor([0.3, 0.6], device=DEV),), ops.differential_attention, ops.differential_attention_backward
        want = fwd(q, k, v, *more, for_backward=True)
        got = fwd(far(q), far(k), far(v), *more, for_backward=True)
        for x, y in zip(got + bwd(far(do), far(q), far(k), far(v), *got, *more), want + bwd(do, q, k, v, *want, *more)):
            assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("Tq,starts", [(1, [0, 100, 37]), (70, [0, 65, -20]), (70, [-70, 230, 31])])
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_keys_behind_the_last_query_of_a_causal_call_are_never_used(maps, Tq, starts):
    """a cache without kv_lens: rows that no query reaches may hold anything, and get zero gradients"""
    ops, Tk = _ops(), 300
    ends = [min(max(s + Tq, 0), Tk) for s in starts]
    q, k, v, do, lens = _inputs(maps, len(starts), Tq, Tk, 4, 2, 64, torch.float16, ends)
    q, k, v, do, lens = (t.to(DEV) for t in (q, k, v, do, lens))
    if maps == 1:
        more = (rnd(4, 32, dtype=torch.float16, seed=9).to(DEV), ops.relative_buckets(32, 128, False, device=DEV))
        fwd, bwd = ops.relative_attention, ops.relative_attention_backward
    else:
        more = (torch.rand(4, generator=torch.Generator().manual_seed(3)).to(DEV),)
        fwd, bwd = ops.differential_attention, ops.differential_attention_backward
    kw = dict(causal=True, q_start=torch.tensor(starts, dtype=torch.int32, device=DEV))
    want = fwd(q, k, v, *more, for_backward=True, kv_lens=lens, **kw)
    got = fwd(q, k, v, *more, for_backward=True, **kw)
    grads = bwd(do, q, k, v, *got, *more, **kw)
    for x, y in zip(got + grads, want + bwd(do, q, k, v, *want, *more, kv_lens=lens, **kw)):
        assert torch.equal(x, y)
        assert not x.isnan().any()
    for b, n in enumerate(ends):
        assert grads[1][b, n:].abs().sum() == 0 and grads[2][b, n:].abs().sum() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("Tq", [1, 90])
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention_of_broadcast_keys(maps, Tq):
    """one sequence's keys and values for all of a batch (stride 0), a broadcast gradient: what copies give"""
    ops, dt = _ops(), torch.bfloat16
    q, k, v, do, _ = (x if x is None else x.to(DEV) for x in _inputs(maps, 3, Tq, 120, 4, 2, 64, dt, None))
    k, v, do = k[:1].expand(3, -1, -1, -1), v[:1].expand(3, -1, -1, -1), do[:1, :1].expand(3, Tq, -1, -1)
    if maps == 1:
        more = (rnd(4, 32, dtype=dt, seed=9).to(DEV), ops.relative_buckets(32, 128, device=DEV))
        fwd, bwd = ops.relative_attention, ops.relative_attention_backward
    else:
        more, fwd, bwd = (torch.tensor([0.3, 0.6, 0.1, 0.9], device=DEV),), ops.differential_attention, ops.differential_attention_backward
    got = fwd(q, k, v, *more, causal=True, for_backward=True)
    want = fwd(q, k.contiguous(), v.contiguous(), *more, causal=True, for_backward=True)
    for x, y in zip(got + bwd(do, q, k, v, *got, *more, causal=True), want + bwd(do.contiguous(), q, k.contiguous(), v.contiguous(), *want, *more, causal=True)):
        assert torch.equal(x, y) and x.is_contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("Tq,Tk,causal", [(90, 90, False), (20, 40, True), (300, 1100, False)])
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_rows_that_see_one_key_have_no_gradient(maps, Tq, Tk, causal):
    """softmax over one key is 1 whatever its score: dq and dk are 0, up to the 32-bit sums of W (2^-16 of its terms' sizes)"""
    ops, dt, d = _ops(), torch.bfloat16, 64
    q, k, v, do, lens = (x.to(DEV) for x in _inputs(maps, 2, Tq, Tk, 2, 2, d, dt, [Tk, 1]))
    if maps == 1:
        more = (rnd(2, 32, dtype=dt, seed=9).to(DEV), ops.relative_buckets(32, 128, device=DEV))
        fwd, bwd = ops.relative_attention, ops.relative_attention_backward
    else:
        more, fwd, bwd = (torch.tensor([0.7, 0.9], device=DEV),), ops.differential_attention, ops.differential_attention_backward
    got = fwd(q, k, v, *more, causal=causal, kv_lens=lens, for_backward=True)
    dq, dk = bwd(do, q, k, v, *got, *more, causal=causal, kv_lens=lens)[:2]
    w = torch.einsum("ihc,hc->ih", do[1].double().abs(), v[1, 0].double().abs()).repeat_interleave(maps, 1)   # (Tq, heads): |dO| |V|
    assert (dq[1].double().abs() <= 2.0 ** -16 * d ** -0.5 * w[..., None] * k[1, 0].double().abs()).all()
    assert (dk[1, 0].double().abs() <= 2.0 ** -16 * d ** -0.5 * torch.einsum("ih,ihc->hc", w, q[1].double().abs())).all()
    assert dk[1, 1:].abs().sum() == 0 and dq[0].abs().max() > 0


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention_scale(maps):
    _check(maps, (1, 90, 90, 2, 2, 64), "fp16", True, scale=0.4)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 200, 230, 2, 2, 64), (2, 7, 230, 4, 2, 40)])
@pytest.mark.parametrize("case", ["one bucket", "own map", "reach 4096", "no reach", "forbidden", "lowest"])
def test_relative_attention_tables(shape, case):
    ops = _ops()
    H = shape[3]
    table, buckets = rnd(H, 32, dtype=torch.float16, seed=9), ops.relative_buckets(32, 128, device="cpu")
    if case == "one bucket":
        table, buckets = table[:, :1].contiguous(), torch.zeros(3, dtype=torch.int32)
    elif case == "own map":          # any map, not monotone; entries outside are clamped
        buckets = torch.randint(0, 32, (2 * 40 + 1,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    elif case == "reach 4096":
        buckets = ops.relative_buckets(32, 4096, device="cpu")
    elif case == "no reach":
        buckets = torch.tensor([5], dtype=torch.int32)
    elif case == "forbidden":        # a bucket of -inf: pairs that are never seen, some rows without any
        table[:, 16:] = -math.inf
        table[0, :] = -math.inf
    elif case == "lowest":           # the type's lowest value outweighs every score
        table[:, 3] = torch.finfo(torch.float16).min
    _check(1, shape, "fp16", extra=(table, buckets), start=[7] * shape[0])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 300, 300, 2, 2, 64), (3, 30, 41, 2, 1, 160), (40, 20, 20, 1, 1, 32)], ids=str)
@pytest.mark.parametrize("n", [64, 65, 200])
def test_relative_attention_of_many_buckets(shape, n):
    table = rnd(shape[3], n, dtype=torch.bfloat16, seed=9)
    buckets = torch.randint(0, n, (2 * 90 + 1,), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    _check(1, shape, "bf16", extra=(table, buckets))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [700, 1500])   # rows whole, and split over workgroups
def test_table_gradient_where_outputs_round_alike(T):
    """values about 1: all outputs round the same way, and so D is off the same way in all rows.  Beyond the bias's reach that has
    to cancel: dtable is off by its own rounding and by what is left of the pairs within reach"""
    ops, H, d, R, u = _ops(), 2, 32, 128, 2.0 ** -8
    q, k = rnd(1, T, H, d, dtype=torch.bfloat16, seed=1), rnd(1, T, H, d, dtype=torch.bfloat16, seed=2)
    v, do = rnd(1, T, H, d, dtype=torch.bfloat16, scale=0.05, shift=1.003, seed=3), rnd(1, T, H, d, dtype=torch.bfloat16, scale=0.1, shift=1.0, seed=4)
    table, buckets = rnd(H, 32, dtype=torch.bfloat16, seed=9), ops.relative_buckets(32, R, device="cpu")
    a = [t.to(DEV) for t in (q, k, v, table, buckets)]
    out, lse = ops.relative_attention(*a, for_backward=True)
    got = ops.relative_attention_backward(do.to(DEV), *a[:3], out, lse, *a[3:])[3].cpu().double()
    Q, K, V, G = (t[0].double().transpose(0, 1) for t in (q, k, v, do))
    rel = torch.arange(T)[None] - torch.arange(T)[:, None]
    b = buckets.long()[rel.clamp(-R, R) + R]
    P = (Q @ K.transpose(1, 2) * d ** -0.5 + table.double()[:, b]).softmax(-1)
    W, O_ = G @ V.transpose(1, 2), P @ V
    D = (G * O_).sum(-1, keepdim=True)
    off = 2 * u * (G.abs() * O_.abs()).sum(-1, keepdim=True)    # of D: out rounded, P rounded (V > 0)
    add = lambda x: torch.stack([torch.zeros(32, dtype=torch.float64).index_add(0, b.flatten(), y.flatten()) for y in x])   # noqa: E731
    want = add(P * (W - D))
    bound = u * want.abs() + add(P * off * (rel.abs() < R)) + 2.0 ** -18 * add(P * (G.abs() @ V.abs().transpose(1, 2) + D.abs()))
    assert ((got - want).abs() <= bound).all(), ((got - want).abs() / bound).max()


@pytest.mark.gpu
def test_relative_attention_clamps_bucket_numbers():
    ops = _ops()
    q, k, v, do, _ = _inputs(1, 1, 40, 40, 2, 2, 64, torch.float16, None)
    table = rnd(2, 8, dtype=torch.float16, seed=9).to(DEV)
    wild = torch.tensor([-1, 3, 8, 1 << 30, -(1 << 31)], dtype=torch.int32, device=DEV)
    tame = torch.tensor([0, 3, 7, 7, 0], dtype=torch.int32, device=DEV)
    a = [t.to(DEV) for t in (q, k, v)]
    res = []
    for b in (wild, tame):
        out, lse = ops.relative_attention(*a, table, b, for_backward=True)
        res.append((out, *ops.relative_attention_backward(do.to(DEV), *a, out, lse, table, b)))
    for x, y in zip(*res):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention_of_a_long_cache(maps):
    """keys whose byte offsets pass 2^32 (a slice of a wide cache) give what the same keys packed give"""
    ops = _ops()
    T, wide, d = 140000, 16384, 64
    cache = torch.zeros((1, T, wide), dtype=torch.float16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    k = cache[..., 128:128 + maps * d].unflatten(-1, (maps, d))
    v = cache[..., wide - maps * d:].unflatten(-1, (1, maps * d))
    k.copy_(torch.randn(k.shape, generator=g, device=DEV))
    v.copy_(torch.randn(v.shape, generator=g, device=DEV))
    for Tq in (1, 40):
        q = torch.randn((1, Tq, maps, d), generator=g, device=DEV).half()
        if maps == 1:
            t, b = torch.randn((1, 32), generator=g, device=DEV).half(), ops.relative_buckets(32, 128)
            f = lambda kk, vv: ops.relative_attention(q, kk, vv, t, b, causal=True)   # noqa: E731
        else:
            lam = torch.tensor([0.4], device=DEV)
            f = lambda kk, vv: ops.differential_attention(q, kk, vv, lam, causal=True)   # noqa: E731
        assert torch.equal(f(k, v), f(k.contiguous(), v.contiguous()))
    del cache, k, v


@pytest.mark.gpu
@pytest.mark.parametrize("shape,lens", [((1, 1, 9001, 1, 1, 64), None), ((1, 2, 36000, 2, 1, 40), None), ((2, 1, 36000, 1, 1, 128), [36000, 130]),
                                        ((1, 40, 20000, 1, 1, 64), [19000])], ids=str)
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention_joined_from_many_parts(maps, shape, lens):
    """few problems with many keys: 17 to more than 64 parts, some of them without keys"""
    _check(maps, shape, "fp16", True, lens, None if lens is None else [n - shape[1] for n in lens], train=False)


@pytest.mark.gpu
@pytest.mark.parametrize("maps", [1, 2], ids=["relative", "differential"])
def test_attention_gradient_against_differences(maps):
    """dq, dk, dv and the learned weights' gradient along a direction against differences of the 64-bit definition"""
    ops = _ops()
    B, T, H, d = 1, 12, 2, 16
    q, k, v, do, _ = _inputs(maps, B, T, T, H, H, d, torch.float16, None)
    a = [t.to(DEV) for t in (q, k, v)]
    buckets = ops.relative_buckets(8, 6, device="cpu")
    w = rnd(H, 8, dtype=torch.float16, seed=9) if maps == 1 else torch.tensor([0.3, 0.7])

    def f(x):
        kw = dict(table=x[3], buckets=buckets) if maps == 1 else dict(lam=x[3])
        return (O.attention(maps, x[0], x[1], x[2], True, **kw)["out"][0] * do.double()).sum().item()
    if maps == 1:
        out, lse = ops.relative_attention(*a, w.to(DEV), buckets.to(DEV), causal=True, for_backward=True)
        got = ops.relative_attention_backward(do.to(DEV), *a, out, lse, w.to(DEV), buckets.to(DEV), causal=True)
    else:
        out, out2, lse = ops.differential_attention(*a, w.to(DEV), causal=True, for_backward=True)
        got = ops.differential_attention_backward(do.to(DEV), *a, out, out2, lse, w.to(DEV), causal=True)
    want = O.attention(maps, q, k, v, True, **(dict(table=w, buckets=buckets) if maps == 1 else dict(lam=w)), dout=do)
    h = 1e-5
    for i, name in enumerate(("dq", "dk", "dv", "dtable" if maps == 1 else "dlam")):
        x = [t.double() for t in (q, k, v, w)]
        step = rnd(*x[i].shape, seed=20 + i).double()
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + h * step, x[i] - h * step
        num = (f(hi) - f(lo)) / (2 * h)
        ana = (got[i].cpu().double() * step).sum().item()
        assert abs(num - ana) <= (want[name][1] * step.abs()).sum().item() + 1e-6 * (1 + abs(num)), name


# ---------------------------------------------------------------------------------------------------------------
# how they are called
# ---------------------------------------------------------------------------------------------------------------
def _layer(ops, x, w):
    """a fused projection's rows through both attentions and back to the projection's gradient: the operators as a layer uses
    them together.  x (B, T, (4 + 2 + 2) 64) fp16: four query heads, two key heads, two value heads"""
    q, k, v = x[..., :256].unflatten(-1, (4, 64)), x[..., 256:384].unflatten(-1, (2, 64)), x[..., 384:].unflatten(-1, (2, 64))
    norm = (w["wq"], w["wk"], w["rope"])
    qn, kn = ops.qk_norm_rope(q, k, *norm)
    out, lse = ops.relative_attention(qn, kn, v, w["table"], w["buckets"], causal=True, for_backward=True)
    # the same heads as two pairs of maps over one head of values
    vd = v.flatten(2).unflatten(-1, (1, 128))
    od, od2, lsed = ops.differential_attention(qn, kn, vd, w["lam"], causal=True, for_backward=True)
    on, _ = ops.qk_norm_rope(od, None, w["wo"], None)            # the norm of each head's difference
    g = w["g"]
    d_od, _, dwo, _ = ops.qk_norm_rope_backward(g.unflatten(-1, (2, 128)), None, od, None, w["wo"], None)
    r = ops.relative_attention_backward(g.unflatten(-1, (4, 64)), qn, kn, v, out, lse, w["table"], w["buckets"], causal=True)
    s = ops.differential_attention_backward(d_od, qn, kn, vd, od, od2, lsed, w["lam"], causal=True)
    dq, dk, dwq, dwk = ops.qk_norm_rope_backward(r[0] + s[0], r[1] + s[1], q, k, *norm)
    return [out, on, dq, dk, r[2] + s[2].reshape(r[2].shape), r[3], s[3], dwq, dwk, dwo]


def _layer_weights(ops, B, T, seed):
    x = rnd(B, T, 512, dtype=torch.float16, seed=seed).to(DEV)
    w = dict(wq=rnd(64, shift=1.0, scale=0.2, seed=1), wk=rnd(64, shift=1.0, scale=0.2, seed=2), wo=rnd(128, shift=1.0, scale=0.2, seed=3),
             rope=ops.rope_table(T, 64, device="cpu"), table=rnd(4, 32, dtype=torch.float16, seed=4),
             buckets=ops.relative_buckets(32, 128, False, device="cpu"), lam=torch.tensor([0.2, 0.6]), g=rnd(B, T, 256, dtype=torch.float16, seed=5))
    return x, {n: t.to(DEV) for n, t in w.items()}


@pytest.mark.gpu
def test_a_layer_of_them_together():
    """forward and backward through all three against the 64-bit chain: each operator within its own bound on the inputs that it
    got (the bounds of a chain's later links count the earlier ones' roundings as given)"""
    ops = _ops()
    x, w = _layer_weights(ops, 2, 150, 11)
    out, on, dq, dk, dv, dtable, dlam, dwq, dwk, dwo = _layer(ops, x, w)
    c = {n: t.cpu() for n, t in w.items()}
    q, k, v = x[..., :256].unflatten(-1, (4, 64)), x[..., 256:384].unflatten(-1, (2, 64)), x[..., 384:].unflatten(-1, (2, 64))
    qn, kn = ops.qk_norm_rope(q, k, w["wq"], w["wk"], w["rope"])
    within(qn, O.head_norm(q.cpu(), c["wq"], c["rope"])["y"], "qn")
    vd = v.flatten(2).unflatten(-1, (1, 128))
    g = c["g"]
    want = O.attention(1, qn.cpu(), kn.cpu(), v.cpu(), True, table=c["table"], buckets=c["buckets"], dout=g.unflatten(-1, (4, 64)))
    within(out, want["out"], "out")
    within(dtable, want["dtable"], "dtable")
    od = ops.differential_attention(qn, kn, vd, w["lam"], causal=True)
    wn = O.head_norm(od.cpu(), c["wo"], dy=g.unflatten(-1, (2, 128)))
    within(on, wn["y"], "on")
    within(dwo, wn["dw"], "dwo")
    d_od = wn["dx"][0].half()
    wd = O.attention(2, qn.cpu(), kn.cpu(), vd.cpu(), True, lam=c["lam"], dout=ops.qk_norm_rope_backward(
        w["g"].unflatten(-1, (2, 128)), None, od, None, w["wo"], None)[0].cpu())
    within(dlam, wd["dlam"], "dlam")
    assert d_od.shape == od.shape
    both = want["dv"][0] + wd["dv"][0].reshape(want["dv"][0].shape)
    within(dv, (both, want["dv"][1] + wd["dv"][1].reshape(both.shape) + 2.0 ** -11 * both.abs() * 3 + 2.0 ** -24), "dv")


@pytest.mark.gpu
def test_equal_calls_give_equal_bits_and_graphs_replay():
    """two captured graphs of the same layer, replayed in turn with eager calls and new inputs between, give the eager bits"""
    ops = _ops()
    x, w = _layer_weights(ops, 2, 150, 11)
    y, _ = _layer_weights(ops, 2, 150, 12)
    eager = [_layer(ops, t, w) for t in (x, y)]
    for a, b in zip(eager[0], _layer(ops, x, w)):
        assert torch.equal(a, b)
    held = [x.clone(), x.clone()]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _layer(ops, held[0], w)
    torch.cuda.current_stream().wait_stream(side)
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_layer(ops, h, w))
        graphs.append(g)
    for turn in range(3):
        for i, g in enumerate(graphs):
            src = (turn + i) % 2
            held[i].copy_((x, y)[src])
            g.replay()
            _layer(ops, (x, y)[1 - src], w)
            torch.cuda.synchronize()
            for a, b in zip(outs[i], eager[src]):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_first_calls_inside_a_capture():
    """a geometry that no call has launched before is captured and replayed like any other"""
    ops = _ops()
    q, k, v, do, _ = _inputs(2, 1, 200, 200, 1, 1, 104, torch.bfloat16, None)
    q, k, v, do, lam = (t.to(DEV) for t in (q, k, v, do, torch.tensor([0.5])))

    def step():
        out, out2, lse = ops.differential_attention(q, k, v, lam, causal=True, for_backward=True)
        return [out, *ops.differential_attention_backward(do, q, k, v, out, out2, lse, lam, causal=True)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = step()
    for _ in range(3):
        for t in held:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_calls_on_other_streams():
    """two streams at once, each with its own workspaces: what one stream alone gives"""
    ops = _ops()
    x, w = _layer_weights(ops, 2, 150, 11)
    y, _ = _layer_weights(ops, 2, 150, 12)
    eager = [_layer(ops, t, w) for t in (x, y)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for t, s in zip((x, y), streams):
        with torch.cuda.stream(s):
            got.append([_layer(ops, t, w) for _ in range(3)])
    torch.cuda.synchronize()
    for e, runs in zip(eager, got):
        for r in runs:
            for a, b in zip(e, r):
                assert torch.equal(a, b)


@pytest.mark.gpu
def test_norm_feeds_reference_attention():
    """normed and rotated heads in the framework's own reference attention: q_alpha carries the scale and log2 e"""
    ops = _ops()
    T, h, d = 256, 8, 40
    q, k, v = (rnd(1, T, h, d, dtype=torch.float16, seed=i) for i in (1, 2, 3))
    w = torch.ones(d)
    rope = ops.rope_table(T, d, device="cpu")
    qn, kn = ops.qk_norm_rope(q.to(DEV), k.to(DEV), w.to(DEV), w.to(DEV), rope.to(DEV), q_alpha=ops.attn_q_alpha(d))
    vt = v.to(DEV).reshape(T, h * d).t().contiguous()
    out = ops.ref_attention(qn.reshape(T, h * d), h * d, kn.reshape(T, h * d), h * d, vt, T, 1, T, h, d, q_log2_scaled=True)
    qo, ko = O.head_norm(q, w, rope)["y"][0], O.head_norm(k, w, rope)["y"][0]
    s = torch.einsum("bihd,bjhd->bhij", qo, ko) * d ** -0.5
    want = torch.einsum("bhij,bjhd->bihd", s.softmax(-1), v.double()).reshape(T, h * d)
    # q, k are rounded once more here: |ds| <= 2 * 2^-11 sum |q||k| scale <= 2^-10 sqrt(d), P's and the output's roundings on top
    bound = (2 * 2.0 ** -10 * d ** 0.5 + 2.0 ** -10) * v.abs().max().double()
    assert (out.cpu().double() - want).abs().max() <= bound


@pytest.mark.gpu
def test_empty_calls():
    ops = _ops()
    e = lambda *s: torch.empty(s, dtype=torch.float16, device=DEV)   # noqa: E731
    t, b = torch.zeros((2, 32), dtype=torch.float16, device=DEV), ops.relative_buckets(32, 128)
    w = torch.ones(64, device=DEV)
    q, k = ops.qk_norm_rope(e(2, 0, 2, 64), e(2, 0, 1, 64), w, w)
    assert q.shape == (2, 0, 2, 64) and k.shape == (2, 0, 1, 64)
    g = ops.qk_norm_rope_backward(q, k, q, k, w, w)
    assert g[2].abs().max() == 0 and g[3].abs().max() == 0
    out, lse = ops.relative_attention(torch.ones_like(e(1, 3, 2, 64)), e(1, 0, 2, 64), e(1, 0, 2, 64), t, b, for_backward=True)
    assert out.shape == (1, 3, 2, 64) and out.abs().max() == 0 and (lse == -math.inf).all()
    r = ops.relative_attention_backward(torch.ones_like(out), torch.ones_like(out), e(1, 0, 2, 64), e(1, 0, 2, 64), out, lse, t, b)
    assert r[0].abs().max() == 0 and r[1].shape == (1, 0, 2, 64) and r[3].abs().max() == 0
    out = ops.differential_attention(e(1, 0, 4, 64), e(1, 5, 4, 64), e(1, 5, 2, 128), torch.ones(2, device=DEV))
    assert out.shape == (1, 0, 2, 128)


@pytest.mark.gpu
@pytest.mark.parametrize("change", ["type of v", "shape of k", "heads", "float table", "table heads", "even buckets", "int64 lens", "lens shape", "channels apart",
                                    "misaligned", "odd strides", "width", "scale", "far reach", "lam type", "pairs"])
def test_wrappers_refuse(change):
    ops = _ops()
    a = dict(q=rnd(2, 8, 4, 64, dtype=torch.float16).to(DEV), k=rnd(2, 8, 2, 64, dtype=torch.float16).to(DEV), v=rnd(2, 8, 2, 64, dtype=torch.float16).to(DEV),
             table=torch.zeros((4, 32), dtype=torch.float16, device=DEV), buckets=ops.relative_buckets(32, 128))
    kw = {}
    if change == "type of v":
        a["v"] = a["v"].bfloat16()
    elif change == "shape of k":
        a["k"] = a["k"][:, :7]
    elif change == "heads":
        a["q"] = a["q"][:, :, :3]
        a["table"] = a["table"][:3].contiguous()
    elif change == "float table":
        a["table"] = a["table"].float()
    elif change == "table heads":
        a["table"] = a["table"][:2].contiguous()
    elif change == "even buckets":
        a["buckets"] = a["buckets"][1:].contiguous()
    elif change == "int64 lens":
        kw["kv_lens"] = torch.tensor([8, 8], device=DEV)
    elif change == "lens shape":
        kw["kv_lens"] = torch.tensor([8], dtype=torch.int32, device=DEV)
    elif change == "channels apart":
        a["k"] = a["k"].transpose(2, 3).contiguous().transpose(2, 3)
    elif change == "misaligned":
        a["q"] = torch.zeros(2 * 8 * 4 * 64 + 1, dtype=torch.float16, device=DEV)[1:].view(2, 8, 4, 64)
    elif change == "odd strides":
        a["q"] = torch.zeros((2, 8, 4, 68), dtype=torch.float16, device=DEV)[..., :64]
    elif change == "width":
        for n in "qkv":
            a[n] = torch.cat([a[n]] * 3, -1)
    elif change == "scale":
        kw["scale"] = -1.0
    elif change == "far reach":
        a["buckets"] = torch.zeros(2 * 4097 + 1, dtype=torch.int32, device=DEV)
    elif change in ("lam type", "pairs"):
        lam = torch.ones(2, device=DEV, dtype=torch.float64 if change == "lam type" else torch.float32)
        with pytest.raises((TypeError, ValueError)):
            ops.differential_attention(a["q"] if change == "lam type" else a["q"][:, :, :3], a["k"], torch.zeros((2, 8, 1, 128), dtype=torch.float16, device=DEV), lam)
        return
    with pytest.raises((TypeError, ValueError)):
        ops.relative_attention(*a.values(), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("change", ["no weight", "weight type", "rope width", "rope rows", "positions alone", "positions type", "k tokens", "width"])
def test_norm_wrapper_refuses(change):
    ops = _ops()
    q, k = rnd(2, 8, 4, 64, dtype=torch.float16).to(DEV), rnd(2, 8, 2, 64, dtype=torch.float16).to(DEV)
    w, rope, kw = torch.ones(64, device=DEV), ops.rope_table(8, 64), {}
    a = dict(q=q, k=k, wq=w, wk=w, rope=rope)
    if change == "no weight":
        a["wk"] = None
    elif change == "weight type":
        a["wq"] = w.half()
    elif change == "rope width":
        a["rope"] = ops.rope_table(8, 72)
    elif change == "rope rows":
        a["rope"] = ops.rope_table(7, 64)
    elif change == "positions alone":
        a["rope"], kw["positions"] = None, torch.zeros((2, 8), dtype=torch.int32, device=DEV)
    elif change == "positions type":
        kw["positions"] = torch.zeros((2, 8), device=DEV, dtype=torch.int64)
    elif change == "k tokens":
        a["k"] = k[:, :7]
    elif change == "width":
        a["q"] = rnd(2, 8, 4, 60, dtype=torch.float16).to(DEV)
    with pytest.raises((TypeError, ValueError)):
        ops.qk_norm_rope(*a.values(), **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("side", [0, 1])
def test_norm_wrapper_refuses_expanded_outputs(side):
    ops = _ops()
    q, w = rnd(2, 8, 4, 64, dtype=torch.float16).to(DEV), torch.ones(64, device=DEV)
    shared = torch.zeros((1, 8, 4, 64), dtype=torch.float16, device=DEV).expand(2, -1, -1, -1)
    with pytest.raises(ValueError, match="expanded"):
        ops.qk_norm_rope(q, q.clone(), w, w, **{("q_out", "k_out")[side]: shared})
    assert shared.abs().max() == 0


@pytest.mark.gpu
def test_profile_counts_the_calls():
    ops = _ops()
    x, w = _layer_weights(ops, 1, 64, 1)
    with ops.profile() as p:
        _layer(ops, x, w)
    names = {k: v["launches"] for k, v in p.result.items()}
    assert names == {"head_norm_kernels": 4, "relative_attention_kernels": 2, "differential_attention_kernels": 2}
    assert p.by_shape is not None
