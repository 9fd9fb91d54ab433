"""Group normalisation, dropout and the gated delta rule at their edges: precision of 16-bit results, long walks of a thread, the scans' wide
form, padding that must have no influence, calls that must be refused.  References are stated in 64 bits on the CPU."""
import pytest
import torch

from test_gpu_operators import DTYPES, delta_inputs, delta_reference, ids

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ precision of 16-bit results
def rounded_once(u, w, what):
    """||u - w|| <= (r + 2^-12) ||w||, r ||w|| the two-norm of w's own rounding to u's type (bf16: r = 2^-9.2).  What is rounded comes from products
    whose operands have at least 16 bits: each factor is off by at most 2^-16 of itself, a product by 3 * 2^-16 with the part of it that is
    left out.  The errors of a sum's terms have either sign and grow as the terms' two-norm, which is at most four times the result's for
    the inputs here: 3 * 4 * 2^-16 < 2^-12."""
    dtype, u, w = u.dtype, u.detach().double().cpu(), w.detach().double()
    once, err = float((w.to(dtype).double() - w).norm() / w.norm()), float((u - w).norm() / w.norm())
    assert err <= once + 2.0 ** -12, (what, err, once)


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=ids)
@pytest.mark.parametrize("T,B,Hk,r,dk,dv", [(40, 2, 2, 1, 64, 128), (200, 1, 1, 2, 128, 72), (70, 9, 16, 1, 16, 72)], ids=str)
@pytest.mark.parametrize("train", [False, True])
def test_delta_output_is_rounded_once(cuda, dtype, T, B, Hk, r, dk, dv, train):
    from speech_amd import ops
    args, _, _ = delta_inputs(T, B, Hk, r, dk, dv, dtype, 11)
    dev = [t.to(cuda).requires_grad_(train) for t in args]
    o, _ = ops.gated_delta_rule(*dev[:5], state=dev[5], normalize=True)
    ro, _ = delta_reference(*(t.double() for t in args), None, dk ** -0.5, True, False)
    rounded_once(o, ro, "o")


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=ids)
@pytest.mark.parametrize("T,B,Hk,r,dk,dv", [(200, 1, 2, 2, 64, 128), (200, 1, 1, 2, 128, 72), (70, 9, 16, 1, 16, 72)], ids=str)
@pytest.mark.parametrize("normalize", [True, False])
def test_delta_gradients_are_rounded_once(cuda, dtype, T, B, Hk, r, dk, dv, normalize):
    from speech_amd import ops
    args, go, gs = delta_inputs(T, B, Hk, r, dk, dv, dtype, 11)
    dev, ref = [t.to(cuda).requires_grad_(True) for t in args], [t.double().requires_grad_(True) for t in args]
    o, final = ops.gated_delta_rule(*dev[:5], state=dev[5], normalize=normalize)
    ro, rf = delta_reference(*ref, None, dk ** -0.5, normalize, False)
    got = torch.autograd.grad([o, final], dev[:3], [go.to(cuda), gs.to(cuda)])
    want = torch.autograd.grad([ro, rf], ref[:3], [go.double(), gs.double()])
    for name, u, w in zip(("dq", "dk", "dv"), got, want):
        rounded_once(u, w, name)


# ------------------------------------------------------------------------------------------ calls that are refused
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_tangents_are_refused(cuda, grad):
    """No operator has a forward-mode derivative: a dual tensor raises, in whichever argument it comes, with and without gradient mode."""
    import torch.autograd.forward_ad as fwd
    from speech_amd import ops
    x, w = torch.randn(4, 6, 16, device=cuda), torch.ones(16, device=cuda)
    q, g = torch.randn(20, 2, 2, 16, device=cuda), -torch.rand(20, 2, 2, device=cuda)
    state, rng = torch.zeros(2, 2, 16, 16, device=cuda), ops.dropout_rng(1, cuda)
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))      # noqa: E731
        calls = [lambda: ops.group_norm(dual(x), w, w, 4), lambda: ops.group_norm(x, dual(w), w, 4), lambda: ops.group_norm(x, w, dual(w), 4),
                 lambda: ops.group_norm(x, w, w, 4, residual=dual(x)), lambda: ops.dropout(dual(x), 0.5, rng), lambda: ops.dropout(x, 0.5, rng, residual=dual(x))]
        for T in (20, 5):
            a = (q[:T], q[:T], q[:T], g[:T], -g[:T], state)
            calls += [lambda a=a, i=i: ops.gated_delta_rule(*(dual(t) if j == i else t for j, t in enumerate(a))) for i in range(6)]
        a = (q[0], q[0], q[0], g[0], -g[0], state)
        calls += [lambda i=i: ops.gated_delta_step(*(dual(t) if j == i else t for j, t in enumerate(a))) for i in range(6)]
        for i, call in enumerate(calls):
            with pytest.raises(NotImplementedError):
                call()
                raise AssertionError(i)
        # what carries no tangent still runs inside the level
        assert torch.isfinite(ops.group_norm(x, w, w, 4)).all() and torch.isfinite(ops.gated_delta_step(*a)).all()


# ------------------------------------------------------------------------------------------ group norm: threads that walk far
@pytest.mark.parametrize("shape", [(1, 30, 1000, 257), (385, 1, 300, 129)], ids=str)
@pytest.mark.parametrize("click,offset", [(1e4, 0.0), (-3e4, 50.0)])
def test_group_norm_click_in_a_long_walk(cuda, shape, click, offset):
    """One channel a group, the first frame of every sample a click: with 257 and 129 channels a workgroup has one row of threads, a thread walks
    469 and 300 positions, and its first one is the click.  The variance is a sum of positive terms in a chain of 118 steps of four positions
    with three roundings each, and rstd halves the relative error: 177 half steps of f32, with fewer than 64 of the merging and the rest 256.
    The mean of a walk: a step rounds a mean of size |offset| + 8 + K / n twice, and an error made after n of N positions reaches the walk's end
    as its share n / N: over 118 steps at most 118 half steps of |offset| + 8 and half a half step of the click K, times the walk's share of
    the sample."""
    from speech_amd import ops
    N, F, T, C = shape
    g = torch.Generator().manual_seed(2)
    x = torch.randn(*shape, generator=g) + offset
    x[:, 0, 0] = click
    w, b = torch.ones(C), torch.zeros(C)
    y = ops.group_norm(x.to(cuda), w.to(cuda), b.to(cuda), C).double().cpu()
    v = x.double()
    m = v.mean((1, 2), keepdim=True)
    rstd = 1 / torch.sqrt(((v - m) ** 2).mean((1, 2), keepdim=True) + 1e-5)
    want = (v - m) * rstd
    walk = 469 / 30000 if N == 1 else 1.0
    bound = 256 * 2.0 ** -24 * want.abs() + 2.0 ** -24 * (128 * (abs(offset) + 8) + abs(click) * walk) * rstd
    assert ((y - want).abs() <= bound).all(), float(((y - want).abs() / want.abs().clamp_min(1e-6)).max())
