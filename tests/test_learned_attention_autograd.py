"""What torch tracks of the attention operators with learned positions: nothing, and so inputs with tracked gradients are refused where
torch is recording; inside an autograd.Function, and without recording, they are plain functions."""
import pytest
import torch
from torch.autograd import forward_ad

DEV = "cuda"


def calls(dev, dtype=torch.float16):
    """{name: (function, tensors whose gradients could be asked for, call)}"""
    from aniportrait_amd import hipops as ops
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g).to(dev, dtype)   # noqa: E731
    f = lambda *s: torch.rand(s, generator=g).to(dev)           # noqa: E731
    q, k, v, table, lam, w = r(1, 8, 4, 64), r(1, 8, 2, 64), r(1, 8, 2, 64), r(4, 32), f(2), f(64)
    vd, buckets, rope = r(1, 8, 1, 128), ops.relative_buckets(32, 128, device=dev), ops.rope_table(8, 64, device=dev)
    out, out2, lse, od = r(1, 8, 4, 64), r(1, 8, 2, 128), f(1, 4, 8), r(1, 8, 2, 128)
    return {
        "qk_norm_rope": (ops.qk_norm_rope, [q, k, w, w.clone(), rope], {}),
        "qk_norm_rope_backward": (ops.qk_norm_rope_backward, [r(1, 8, 4, 64), r(1, 8, 2, 64), q, k, w, w.clone(), rope], {}),
        "relative_attention": (ops.relative_attention, [q, k, v, table, buckets], {}),
        "relative_attention_backward": (ops.relative_attention_backward, [r(1, 8, 4, 64), q, k, v, out, lse, table, buckets], {}),
        "differential_attention": (ops.differential_attention, [q, k, vd, lam], {}),
        "differential_attention_backward": (ops.differential_attention_backward, [od.clone(), q, k, vd, od, out2, lse, lam], {}),
    }


NAMES = ["qk_norm_rope", "qk_norm_rope_backward", "relative_attention", "relative_attention_backward", "differential_attention",
         "differential_attention_backward"]


@pytest.mark.parametrize("name", NAMES)
def test_tracked_inputs_are_refused(name):
    """ahead of everything else, so that no GPU is needed"""
    fn, args, kw = calls("cpu")[name]
    for i, t in enumerate(args):
        if not t.is_floating_point():
            continue
        bad = list(args)
        bad[i] = t.clone().requires_grad_()
        with pytest.raises(RuntimeError, match=name + ": an input requires a gradient"):
            fn(*bad, **kw)
        bad[i] = bad[i] * 1                      # not a leaf
        with pytest.raises(RuntimeError, match="requires a gradient"):
            fn(*bad, **kw)
        from aniportrait_amd import hipops as ops
        with torch.no_grad(), pytest.raises(ops.L.HipLibraryError):
            fn(*bad, **kw)                       # on to the next check
        with forward_ad.dual_level():
            bad[i] = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="tangent"):
                fn(*bad, **kw)


def test_tracked_outputs_are_refused():
    fn, args, _ = calls("cpu")["qk_norm_rope"]
    for name in ("q_out", "k_out"):
        with pytest.raises(RuntimeError, match="requires a gradient"):
            fn(*args, **{name: (args[0] if name == "q_out" else args[1]).clone().requires_grad_()})


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_parameters_without_recording(name):
    fn, args, kw = calls(DEV)[name]
    want = fn(*args, **kw)
    with torch.no_grad():
        got = fn(*[t.clone().requires_grad_() if t.is_floating_point() else t for t in args], **kw)
    for a, b in zip(want if isinstance(want, tuple) else (want,), got if isinstance(got, tuple) else (got,)):
        assert torch.equal(a, b) and not b.requires_grad


@pytest.mark.gpu
def test_inside_a_function():
    """the way a training program calls them: gradients arrive at the leaves, and a second derivative is refused, not dropped"""
    from aniportrait_amd import hipops as ops
    _, (q, k, v, table, buckets), _ = calls(DEV)["relative_attention"]

    class Attention(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, table):
            out, lse = ops.relative_attention(q, k, v, table, buckets, causal=True, for_backward=True)
            ctx.save_for_backward(q, k, v, out, lse, table)
            return out

        @staticmethod
        def backward(ctx, dout):
            q, k, v, out, lse, table = ctx.saved_tensors
            return ops.relative_attention_backward(dout, q, k, v, out, lse, table, buckets, causal=True)

    leaves = [t.clone().requires_grad_() for t in (q, k, v, table)]
    y = Attention.apply(*leaves)
    dout = torch.randn(y.shape, generator=torch.Generator().manual_seed(2)).to(DEV, y.dtype)
    got = torch.autograd.grad(y, leaves, dout, retain_graph=True)
    out, lse = ops.relative_attention(q, k, v, table, buckets, causal=True, for_backward=True)
    for a, b in zip(got, ops.relative_attention_backward(dout, q, k, v, out, lse, table, buckets, causal=True)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        torch.autograd.grad(y, leaves, dout, create_graph=True)
