"""Group normalisation with an activation, counter-based dropout and the gated delta rule on the GPU, against plain statements in 64 bits
computed on the CPU.

Tolerances.  A result of type t that is computed in f32 and rounded once is off by at most half a step, eps(t) / 2 of its value (f32: 2^-24,
f16: 2^-11, bf16: 2^-8), plus what the f32 arithmetic before it loses.  That is bounded by D roundings of half an f32 step each on
intermediate values of the size of the result's largest terms `scale`: D * 2^-24 * scale.  Sums over n values run in trees or short chains
and lose at most (chain + log2 n) half steps; the numbers D below count each operator's longest path and are rounded up to a power of two.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ids = lambda t: str(t).replace("torch.", "")      # noqa: E731


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, scale, depth, dtype=None, what=""):
    """|got - want| <= half a step of got's type relative to the value + depth f32 half steps of `scale`."""
    dtype = dtype or got.dtype
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    bound = half_step(dtype) * want.abs() * (1 + 2.0 ** -7) + depth * 2.0 ** -24 * scale + (2.0 ** -25 if dtype == torch.float16 else 0)
    worst = ((got - want).abs() - bound).max() if got.numel() else torch.tensor(-1.0)
    assert worst <= 0, (what, float((got - want).abs().max()), float(scale))


# ------------------------------------------------------------------------------------------ group norm
def gn_reference(x, w, b, G, act, res, lengths, eps=1e-5):
    """x [N,F,T,C] f64, differentiable."""
    N, F, T, C = x.shape
    out = []
    for n in range(N):
        L = T if lengths is None else int(lengths[n])
        xs = x[n, :, :L]
        if xs.numel() == 0:
            out.append(x[n] * 0 + 0 * w + 0 * b + (0 if res is None else res[n] * 0))
            continue
        v = xs.reshape(F, L, G, C // G)
        m = v.mean((0, 1, 3), keepdim=True)
        var = ((v - m) ** 2).mean((0, 1, 3), keepdim=True)
        z = ((v - m) / torch.sqrt(var + eps)).reshape(F, L, C) * w + b
        if res is not None:
            z = z + res[n, :, :L]
        z = torch.relu(z) if act == "relu" else z * torch.sigmoid(z) if act == "silu" else z
        out.append(torch.cat([z, z.new_zeros(F, T - L, C)], 1))
    return torch.stack(out)


def gn_inputs(shape, dtype, seed=0, res=False, offset=0.0):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(*shape, generator=g) * 1.5 + torch.randn(C, generator=g) + offset).to(dtype)
    w, b = 1 + 0.3 * torch.randn(C, generator=g), 0.3 * torch.randn(C, generator=g)
    r = torch.randn(*shape, generator=g).to(dtype) if res else None
    gy = torch.randn(*shape, generator=g).to(dtype)
    return x, w, b, r, gy


GN_SHAPES = [  # N, F, T, C, G: vector widths 8 / 4 / 2 / 1, groups inside, across and as large as a vector, more channels than a workgroup has threads
    (2, 3, 5, 32, 8), (3, 1, 1, 64, 4), (1, 4, 33, 20, 5), (2, 2, 9, 48, 4), (1, 1, 130, 6, 3), (2, 1, 7, 5, 5), (1, 2, 3, 1030, 2),
    (2, 1, 4, 2048, 1), (37, 1, 1, 1024, 8), (5, 1, 1, 2048, 1), (3, 1, 1, 7, 1), (4, 1, 1, 515, 5), (1, 40, 70, 32, 32), (130, 1, 2, 8, 2),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape", GN_SHAPES, ids=str)
@pytest.mark.parametrize("act,res", [("none", False), ("silu", True), ("relu", True), ("relu", False)])
def test_group_norm(cuda, shape, dtype, act, res):
    from speech_amd import ops
    *s, G = shape
    x, w, b, r, gy = gn_inputs(s, dtype, res=res)
    xd, wd, bd = (t.to(cuda).requires_grad_(True) for t in (x, w, b))
    rd = r.to(cuda).requires_grad_(True) if res else None
    y = ops.group_norm(xd, wd, bd, G, act=act, residual=rd)
    x64, w64, b64 = (t.double().requires_grad_(True) for t in (x, w, b))
    r64 = r.double().requires_grad_(True) if res else None
    ref = gn_reference(x64, w64, b64, G, act, r64, None)
    n = s[1] * s[2] * (s[3] // G)
    # xhat loses the mean's and rstd's error (chains of up to kU positions in registers, trees: < 64 half steps with n below 2^17 values) on
    # values up to max |xhat|, gamma, beta, the residual and the activation a few more
    scale = float(ref.detach().abs().max()) + 8
    close(y, ref, scale, 128, what="y")
    pre = gn_reference(x64, w64, b64, G, "none", r64, None).detach()
    leaves = [xd, wd, bd] + ([rd] if res else [])
    gyd = gy.to(cuda)
    if act == "relu":      # where the pre-activation is within the f32 error of zero either branch is right: no gradient is sent there
        keep = (pre.abs() > 128 * 2.0 ** -24 * scale)
        gy = gy * keep
        gyd = gy.to(cuda)
    got = torch.autograd.grad(y, leaves, gyd)
    want = torch.autograd.grad(ref, [x64, w64, b64] + ([r64] if res else []), gy.double())
    # dx = rstd (gamma g - mean - xhat mean): terms up to max |want| and rstd * max |gamma gy|; rstd is at most eps^-1/2 where a group has
    # one value only
    rstd = 1e-5 ** -0.5 if n == 1 else float(_rstd(x, G).max())
    terms = rstd * float(gy.abs().max()) * float(w.abs().max()) * (2 + 4)
    close(got[0], want[0], terms, 256, what="dx")
    # channel sums: N F T terms of size |gy xhat| <= 6 * 5, in chains of a few hundred and trees
    m = s[0] * s[1] * s[2]
    big = float(gy.abs().max()) * 8 * math.sqrt(m)
    close(got[1], want[1], big + float(want[1].abs().max()), 256, torch.float32, "dgamma")
    close(got[2], want[2], big + float(want[2].abs().max()), 256, torch.float32, "dbeta")
    if res:
        close(got[3], want[3], float(gy.abs().max()) * 2, 64, what="dres")


def _rstd(x, G):
    N, F, T, C = x.shape
    v = x.double().view(N, F * T, G, C // G).permute(0, 2, 1, 3).reshape(N, G, -1)
    return 1 / torch.sqrt(v.var(-1, unbiased=False) + 1e-5)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("lengths", [[5, 0, 9, 1], [9, 9, 9, 9], [0, 0, 0, 0], [20, -3, 4, 9]], ids=str)
def test_group_norm_ragged(cuda, dtype, lengths):
    """Frames behind an utterance's end hold NaN and infinities: they are not counted, not read, come out and back as zeros."""
    from speech_amd import ops
    x, w, b, r, gy = gn_inputs((4, 3, 9, 32), dtype, 3, True)
    L = [min(max(v, 0), 9) for v in lengths]
    for n, v in enumerate(L):
        for t in (x, r, gy):
            t[n, :, v:] = float("nan")
            t[n, :, v:, ::2] = float("inf")
    clean = [torch.stack([torch.cat([t[n, :, :v], torch.zeros_like(t[n, :, v:])], 1) for n, v in enumerate(L)]) for t in (x, r, gy)]
    xd, wd, bd, rd = (t.to(cuda).requires_grad_(True) for t in (x, w, b, r))
    y = ops.group_norm(xd, wd, bd, 8, act="silu", residual=rd, lengths=torch.tensor(lengths, device=cuda))
    x64, w64, b64, r64 = (t.double().requires_grad_(True) for t in (clean[0], w, b, clean[1]))
    ref = gn_reference(x64, w64, b64, 8, "silu", r64, L)
    close(y, ref, float(ref.detach().abs().max()) + 8, 128)
    got = torch.autograd.grad(y, [xd, wd, bd, rd], gy.to(cuda))
    want = torch.autograd.grad(ref, [x64, w64, b64, r64], clean[2].double())
    for name, u, v in zip(("dx", "dgamma", "dbeta", "dres"), got, want):
        close(u, v, 60.0, 256, what=name)
    for n, v in enumerate(L):
        assert not y[n, :, v:].any() and not got[0][n, :, v:].any() and not got[3][n, :, v:].any()


def test_group_norm_one_position_ragged(cuda):
    from speech_amd import ops
    x, w, b, r, gy = gn_inputs((6, 1, 1, 64), torch.float32, 4, True)
    L = [1, 0, 1, 0, 1, 1]
    xd, wd, bd, rd = (t.to(cuda).requires_grad_(True) for t in (x, w, b, r))
    y = ops.group_norm(xd, wd, bd, 4, act="silu", residual=rd, lengths=torch.tensor(L, device=cuda))
    x64, w64, b64, r64 = (t.double().requires_grad_(True) for t in (x, w, b, r))
    ref = gn_reference(x64, w64, b64, 4, "silu", r64, L)
    close(y, ref, 10.0, 128)
    for u, v in zip(torch.autograd.grad(y, [xd, wd, bd, rd], gy.to(cuda)), torch.autograd.grad(ref, [x64, w64, b64, r64], gy.double())):
        close(u, v, 60.0, 256)


def test_group_norm_large_mean_and_click(cuda):
    """Statistics are taken around each thread's own values: a mean 1000 times the spread and a click in the first frame keep their digits."""
    from speech_amd import ops
    x, w, b, _, _ = gn_inputs((2, 4, 300, 32), torch.float32, 5)
    x = x * 0.5 + 1000.0
    ref = gn_reference(x.double(), w.double(), b.double(), 8, "none", None, None)
    y = ops.group_norm(x.to(cuda), w.to(cuda), b.to(cuda), 8)
    # x itself is exact; x - mean loses half a step of 1000 (2^-24 * 1000), 2 / 0.5 of that after rstd, and the mean as much again
    close(y, ref, 1000.0 * 4, 16)
    x = x - 1000.0
    x[0, 0, 0] = 1e4
    ref = gn_reference(x.double(), w.double(), b.double(), 8, "none", None, None)
    y = ops.group_norm(x.to(cuda), w.to(cuda), b.to(cuda), 8)
    # the click is xhat ~ sqrt(n) = 70 in its own group; the thread that saw it sums up to (hi - lo) / rows values around it, each losing
    # half a step of 1e4^2: relative to the group's M2 = 1e8 that is at most 64 half steps
    close(y, ref, float(ref.abs().max()), 256)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
def test_group_norm_strides(cuda, dtype):
    """Views are taken as they are: bands cut out, frames reversed in memory order, an odd first element, a time-major result; the same
    values as on contiguous copies, bit for bit where the vector width is the same."""
    from speech_amd import ops
    big = torch.randn(3, 7, 11, 72, device=cuda).to(dtype)
    w, b = torch.rand(32, device=cuda) + 0.5, torch.randn(32, device=cuda)
    for v in (big[:, 1:6, 2:9, 8:40], big.transpose(1, 2)[:, :5, :, 16:48], big[::2, :, :, 3:35], big.permute(2, 1, 0, 3)[..., :32], big[:, :1].expand(3, 4, 11, 72)[..., :32]):
        res = v.flip(0)
        y = ops.group_norm(v, w, b, 4, act="silu", residual=res)
        z = ops.group_norm(v.contiguous(), w, b, 4, act="silu", residual=res.contiguous())
        close(y, z, 10.0, 64)
        t = ops.group_norm(v, w, b, 4, act="silu", residual=res, time_major=True)
        assert t.permute(2, 0, 1, 3).is_contiguous() and torch.equal(t, y)
    # gradients through views, an expanded gradient among them
    v = big[:, 1:6, 2:9, 8:40].detach().requires_grad_(True)
    c = v.detach().contiguous().requires_grad_(True)
    ops.group_norm(v, w, b, 4, time_major=True).float().sum().backward()
    ops.group_norm(c, w, b, 4).float().sum().backward()
    assert torch.equal(v.grad, c.grad)
    x2, x3 = torch.randn(50, 64, device=cuda), torch.randn(5, 10, 64, device=cuda)
    w, b = torch.ones(64, device=cuda), torch.zeros(64, device=cuda)
    assert ops.group_norm(x2, w, b, 4).shape == x2.shape
    assert torch.equal(ops.group_norm(x3, w, b, 4), ops.group_norm(x3[:, None], w, b, 4)[:, 0])
    assert ops.group_norm(x2[:0], w, b, 4).shape == (0, 64)
    e = x2[:0].clone().requires_grad_(True)
    wg = w.clone().requires_grad_(True)
    ops.group_norm(e, wg, b, 4).sum().backward()
    assert not wg.grad.any()


def test_group_norm_repeats_bit_for_bit(cuda):
    from speech_amd import ops
    x, w, b, r, gy = (t.to(cuda) for t in gn_inputs((8, 40, 90, 32), torch.bfloat16, 6, True))
    first = None
    for _ in range(3):
        xs = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        y = ops.group_norm(xs[0], xs[1], xs[2], 8, act="silu", residual=xs[3])
        out = [y.detach(), *torch.autograd.grad(y, xs, gy)]
        first = first or out
        assert all(torch.equal(u, v) for u, v in zip(out, first))


def test_group_norm_refuses(cuda):
    from speech_amd import ops
    x, w = torch.zeros(2, 3, 8, device=cuda), torch.ones(8, device=cuda)
    for kw, text in [(dict(groups=3), "groups"), (dict(act="gelu"), "act"), (dict(residual=x[:1]), "residual"), (dict(residual=x.half()), "residual"),
                     (dict(lengths=torch.ones(3, dtype=torch.int64, device=cuda)), "lengths"), (dict(lengths=torch.ones(2, device=cuda)), "lengths"),
                     (dict(lengths=torch.ones(2, dtype=torch.bool, device=cuda)), "lengths"), (dict(lengths=torch.ones(2, dtype=torch.int64)), "lengths is on"), (dict(weight=w[:4]), "weight"), (dict(x=x.int()), "float"),
                     (dict(x=x[0, 0]), "must be"), (dict(bias=w.cpu()), "bias is on")]:
        a = dict(x=x, weight=w, bias=w, groups=2)
        a.update(kw)
        with pytest.raises(ValueError, match=text):
            ops.group_norm(**a)
    y = ops.group_norm(x.requires_grad_(True), w, w, 2)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


# ------------------------------------------------------------------------------------------ dropout
def philox_draws(n, seed, step, site):
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    at = np.arange((n + 7) // 8, dtype=u)
    c = [at & low, at >> half, np.full_like(at, step & 0xFFFFFFFF), np.full_like(at, site)]
    for r in range(10):
        k0, k1 = u((seed + r * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = u(0xD2511F53) * c[0], u(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ k0, b & low, (a >> half) ^ c[3] ^ k1, a & low]
    return torch.from_numpy(np.stack(c, -1).astype("<u4").view("<u2").reshape(-1)[:n].astype(np.int64))


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("shape,shared", [((1,), False), ((7,), False), ((8, 8), False), ((5, 3, 13), False), ((5, 3, 13), True), ((40, 2, 128), True),
                                          ((1, 9), True), ((300, 1000), False), ((4100, 24), True)], ids=str)
@pytest.mark.parametrize("p,res", [(0.0, False), (0.1, True), (0.5, False), (0.999, True), (1.0, True)])
def test_dropout(cuda, shape, shared, dtype, p, res):
    """The mask is the generator's, element by element, forward and backward; kept values are rounded once, dropped ones exactly zero."""
    from speech_amd import ops
    g = torch.Generator().manual_seed(1)
    x, gy = torch.randn(*shape, generator=g).to(dtype), torch.randn(*shape, generator=g).to(dtype)
    r = torch.randn(*shape, generator=g).to(dtype) if res else None
    seed, step, site = 0x1234567890ABCDEF, 77, 5
    rng = ops.dropout_rng(seed, cuda, step)
    xd = x.to(cuda).requires_grad_(True)
    rd = r.to(cuda).requires_grad_(True) if res else None
    y = ops.dropout(xd, p, rng, site, residual=rd, shared=shared)
    n = x[0].numel() if shared else x.numel()
    thr = int(round(p * 65536))
    keep = (philox_draws(n, seed, step, site) >= thr).view(x.shape[1:] if shared else x.shape).expand(x.shape)
    scale = 65536 / (65536 - thr) if thr < 65536 else 0.0
    want = torch.where(keep, x.double() * scale, 0.0) + (r.double() if res else 0.0)
    close(y, want, float(want.abs().max()) + scale * 6, 4)        # the scale, the product and the sum round in f32
    if not res:
        assert not y.detach().cpu()[~keep].any()
    rng[1] += 1                                                    # the backward belongs to the step the forward used
    got = torch.autograd.grad(y, [xd] + ([rd] if res else []), gy.to(cuda))
    close(got[0], torch.where(keep, gy.double() * scale, 0.0), scale * 6, 4)
    assert not got[0].cpu()[~keep].any()
    if res:
        assert torch.equal(got[1].cpu(), gy)


def test_dropout_values_and_rates(cuda):
    from speech_amd import ops
    x = torch.full((1 << 20,), float("inf"), device=cuda)
    x[::2] = float("nan")
    rng = ops.dropout_rng(3, cuda)
    y = ops.dropout(x, 0.3, rng)
    dropped = y == 0
    # 2^20 draws at p = 0.3: the count's standard deviation is 469; six of them
    assert abs(int(dropped.sum()) - round(0.3 * (1 << 20))) < 6 * 470
    assert torch.isinf(y[1::2][~dropped[1::2]]).all() and torch.isnan(y[::2][~dropped[::2]]).all()
    one = torch.ones(1 << 20, device=cuda)
    masks = [ops.dropout(one, 0.5, ops.dropout_rng(*k), s) > 0 for k, s in (((3, cuda), 0), ((3, cuda), 1), ((4, cuda), 0), ((3, cuda, 1), 0), ((3 + (1 << 40), cuda), 0))]
    for i in range(len(masks)):
        for j in range(i):      # independent masks agree in half of the places: 512 is one standard deviation of 2^20 coins
            assert abs(int((masks[i] == masks[j]).sum()) - (1 << 19)) < 6 * 512
    assert torch.equal(ops.dropout(one, 0.5, ops.dropout_rng(3, cuda), 0), ops.dropout(one, 0.5, ops.dropout_rng(3, cuda), 0))
    # the element's draw does not depend on the tensor it stands in
    assert torch.equal(ops.dropout(one, 0.5, rng)[:1000], ops.dropout(one[:1000], 0.5, rng))


def test_dropout_views_and_refusals(cuda):
    from speech_amd import ops
    rng = ops.dropout_rng(9, cuda)
    big = torch.randn(6, 10, 20, device=cuda)
    for v in (big[:, ::2], big.transpose(0, 2), big[1:, 3:, 5:], big[0, 0, 3:]):
        assert torch.equal(ops.dropout(v, 0.4, rng), ops.dropout(v.contiguous().clone(), 0.4, rng))
    for dt in DTYPES:      # odd first elements: every address alignment of the element
        base = torch.randn(4099, device=cuda).to(dt)
        for o in range(1, 9):
            assert torch.equal(ops.dropout(base[o:], 0.4, rng), ops.dropout(base[o:].clone(), 0.4, rng))
    assert ops.dropout(big[:0], 0.4, rng).shape == (0, 10, 20) and ops.dropout(big[:0], 0.4, rng, shared=True).shape == (0, 10, 20)
    for kw, text in [(dict(p=1.1), "p must"), (dict(p=-0.1), "p must"), (dict(rng=rng.int()), "rng"), (dict(rng=rng[:1]), "rng"), (dict(rng=5), "rng"),
                     (dict(rng=rng.cpu()), "rng is on"), (dict(site=-1), "site"), (dict(residual=big[:1]), "residual"), (dict(x=big[0, 0], shared=True), "shared"),
                     (dict(x=big.long()), "float")]:
        a = dict(x=big, p=0.1, rng=rng)
        a.update(kw)
        with pytest.raises(ValueError, match=text):
            ops.dropout(**a)
    x = big.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(ops.dropout(x, 0.1, rng).sum(), x, create_graph=True)


# ------------------------------------------------------------------------------------------ gated delta rule
def delta_reference(q, k, v, g, beta, state, lengths, scale, normalize, bidirectional):
    """Frame by frame in f64, differentiable; [T,B,H,d]."""
    T, B, Hk, dk = q.shape
    H, dv = v.shape[2:]
    r = H // Hk
    if normalize:
        q, k = (t / torch.sqrt((t * t).sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    q = q * scale
    o = [[None] * B for _ in range(T)]
    final = []
    for b in range(B):
        L = T if lengths is None else min(max(int(lengths[b]), 0), T)
        heads = []
        for h in range(H):
            S = state[b, h] if state is not None else v.new_zeros(dk, dv)
            back = bidirectional and 2 * h >= H
            out = {}
            for t in (range(L - 1, -1, -1) if back else range(L)):
                kt, qt = k[t, b, h // r], q[t, b, h // r]
                S = torch.exp(g[t, b, h]) * S
                u = beta[t, b, h] * (v[t, b, h] - S.t() @ kt)
                S = S + kt[:, None] * u[None, :]
                out[t] = S.t() @ qt
            heads.append(torch.stack([out[t] if t < L else v.new_zeros(dv) for t in range(T)]) if T else v.new_zeros(0, dv))
            final.append(S)
        for t in range(T):
            o[t][b] = torch.stack([x[t] for x in heads])
    return torch.stack([torch.stack(x) for x in o]), torch.stack(final).view(B, H, dk, dv)


def delta_inputs(T, B, Hk, r, dk, dv, dtype, seed=0, state=True, unit=True):
    g = torch.Generator().manual_seed(seed)
    H = Hk * r
    q, k, v = (torch.randn(T, B, n, d, generator=g) for n, d in ((Hk, dk), (Hk, dk), (H, dv)))
    if unit:
        q, k = q / q.norm(dim=-1, keepdim=True), k / k.norm(dim=-1, keepdim=True)
    gg = -torch.exp(torch.empty(H).uniform_(math.log(0.005), 0.0, generator=g)) * torch.nn.functional.softplus(torch.randn(T, B, H, generator=g))
    beta = torch.sigmoid(torch.randn(T, B, H, generator=g))
    s = torch.randn(B, H, dk, dv, generator=g) * 0.3 if state else None
    go, gs = torch.randn(T, B, H, dv, generator=g).to(dtype), 0.1 * torch.randn(B, H, dk, dv, generator=g)
    return [q.to(dtype), k.to(dtype), v.to(dtype), gg, beta, s], go, gs


def delta_check(cuda, args, go, gs, lengths=None, scale=None, normalize=False, bidirectional=False, train=True, dirty=None):
    """Outputs and gradients against the reference.  The two-norm of the difference over the result's, because an element of a recurrence
    has no scale of its own: a 32-bit result is a chain of products of exact f32 splits (the part that is cut off is below 2^-24 of each
    factor) with about sqrt(T) accumulations, 2^-24 * 64 covers it; a 16-bit result adds its own rounding (half a step: eps / 2) and, for o,
    dq and dk, at most two operands cut to 16 bits (2^-16) or rounded to the type (eps / 2 each)."""
    from speech_amd import ops
    dtype = args[0].dtype
    dev = [t.to(cuda).requires_grad_(train) if t is not None else None for t in (dirty or args)]
    L = torch.tensor(lengths, device=cuda) if lengths is not None else None
    o, final = ops.gated_delta_rule(*dev[:5], state=dev[5], lengths=L, scale=scale, normalize=normalize, bidirectional=bidirectional)
    ref = [t.double().requires_grad_(train) if t is not None else None for t in args]
    ro, rf = delta_reference(*ref, lengths, args[0].shape[-1] ** -0.5 if scale is None else scale, normalize, bidirectional)
    assert o.dtype == dtype and final.dtype == torch.float32

    def rel(u, v):
        u, v = u.detach().double().cpu(), v.detach().double()
        assert torch.isfinite(u).all()
        return float((u - v).norm() / v.norm()) if v.norm() > 0 else float(u.norm())
    f32, own = 64 * 2.0 ** -24, half_step(dtype)
    assert rel(o, ro) <= f32 + (3 * own if dtype != torch.float32 else 0), ("o", rel(o, ro))
    assert rel(final, rf) <= f32, ("final", rel(final, rf))
    if not train:
        return o, final
    gd, sd = go.to(cuda), gs.to(cuda)
    got = torch.autograd.grad([o, final], [t for t in dev if t is not None], [gd, sd])
    clean = go.double()
    if lengths is not None:
        for b, n in enumerate(lengths):
            clean[max(min(n, clean.shape[0]), 0):, b] = 0
    want = torch.autograd.grad([ro, rf], [t for t in ref if t is not None], [clean, gs.double()], allow_unused=True)
    want = [torch.zeros_like(t, dtype=torch.float64, device="cpu") if w is None else w for w, t in zip(want, got)]
    for name, u, w in zip(("dq", "dk", "dv", "dg", "dbeta", "dstate"), got, want):
        loose = 3 * own if u.dtype != torch.float32 else 0
        assert rel(u, w) <= 4 * f32 + loose, (name, rel(u, w))
    return o, final, got


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("T", [1, 2, 63, 64, 65, 130])
def test_delta_lengths_of_time(cuda, T, dtype):
    args, go, gs = delta_inputs(T, 2, 2, 1, 16, 24, dtype, T)
    delta_check(cuda, args, go, gs)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dk,dv", [(8, 8), (8, 128), (128, 8), (64, 64), (72, 40), (128, 128), (40, 72)], ids=str)
def test_delta_widths(cuda, dk, dv, dtype):
    args, go, gs = delta_inputs(70, 1, 1, 2, dk, dv, dtype, dk + dv)
    delta_check(cuda, args, go, gs, normalize=True)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("normalize,bidirectional,state", [(True, True, True), (True, False, False), (False, True, False)])
def test_delta_ragged_shared_heads(cuda, dtype, normalize, bidirectional, state):
    """Utterances of length 0, 1, a whole chunk and in between; what lies behind an end is NaN and infinity."""
    args, go, gs = delta_inputs(90, 5, 2, 3, 24, 40, dtype, 3, state, unit=not normalize)
    lengths = [90, 0, 64, 1, 71]
    dirty = [t.clone() if t is not None else None for t in args]
    for b, n in enumerate(lengths):
        for t in dirty[:5]:
            t[n:, b] = float("nan")
        go[n:, b] = float("inf")
    o, final, got = delta_check(cuda, args, go, gs, lengths, None, normalize, bidirectional, dirty=dirty)
    for b, n in enumerate(lengths):
        assert not o[n:, b].any() and not any(x[n:, b].any() for x in got[:5])
    if state:
        assert torch.equal(final[1].cpu(), args[5][1]) and torch.equal(got[5][1].cpu(), gs[1])
    else:
        assert not final[1].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("T", [1, 7, 12, 13, 32, 33, 100])
def test_delta_inference_forms_agree(cuda, T, dtype):
    """Up to 12 frames run the recurrent kernel, more the chunked one; ragged, both directions."""
    args, go, gs = delta_inputs(T, 4, 2, 2, 40, 56, dtype, T)
    delta_check(cuda, args, go, gs, [T, 0, T // 2, 1], normalize=True, bidirectional=True, train=False)


def test_delta_many_chunks_and_workgroups(cuda):
    """1000 frames (the state walks 16 chunks) and more heads than the scans' narrow form takes."""
    args, go, gs = delta_inputs(1000, 1, 1, 1, 16, 32, torch.float32, 8)
    delta_check(cuda, args, go, gs, normalize=True)
    args, go, gs = delta_inputs(66, 48, 4, 1, 8, 72, torch.bfloat16, 9)
    delta_check(cuda, args, go, gs, normalize=True, bidirectional=True)


@pytest.mark.parametrize("T", [5, 80])
def test_delta_gates(cuda, T):
    """beta = 0 (nothing is written), beta = 1, g = 0 (nothing is forgotten), g = -inf and -1e4 (everything is): the gradients stay finite,
    a decay of zero has gradient zero up to the sums' rounding."""
    args, go, gs = delta_inputs(T, 1, 4, 1, 16, 16, torch.float32, 4)
    g, beta = args[3], args[4]
    beta[:, :, 0] = 0.0
    beta[:, :, 1] = 1.0
    g[:, :, 1] = 0.0
    g[::3, :, 2] = -1e4
    ref = [t.clone() for t in args]
    ref[3][::7, :, 3] = -1e4
    g[::7, :, 3] = float("-inf")
    delta_check(cuda, ref, go, gs, dirty=args)
    delta_check(cuda, ref, go, gs, dirty=args, train=False)


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_delta_first_decay_without_a_state(cuda, dtype):
    """The first frame of every walk meets no state: its decay's gradient is exactly zero, in both directions and for every length."""
    from speech_amd import ops
    lengths = [1, 70, 64, 0]
    args, go, gs = delta_inputs(70, 4, 2, 2, 24, 40, dtype, 4, state=False)
    xs = [t.to(cuda).requires_grad_(True) for t in args[:5]]
    o, f = ops.gated_delta_rule(*xs, lengths=torch.tensor(lengths, device=cuda), bidirectional=True)
    gg = torch.autograd.grad([o, f], xs, [go.to(cuda), gs.to(cuda)])[3]
    for b, n in enumerate(lengths):
        if n:
            assert not gg[0, b, :2].any() and not gg[n - 1, b, 2:].any()
        if n > 1:
            assert gg[1:n, b, :2].all() and gg[:n - 1, b, 2:].all()


def test_delta_zero_rows_and_scale(cuda):
    args, go, gs = delta_inputs(70, 2, 2, 1, 16, 16, torch.float32, 5)
    args[0][::5] = 0
    args[1][::4] = 0
    delta_check(cuda, args, go, gs, normalize=True, scale=-0.7)
    delta_check(cuda, args, go, gs, scale=3.0)


def test_delta_gradients_against_differences(cuda):
    """Directional derivatives of the f32 kernels themselves: (L(x + h d) - L(x - h d)) / 2h.  With h = 2^-6 the quotient's truncation error
    is h^2 / 6 of a third derivative, and rounding is 2^-24 sqrt(n) / h: both below 2e-3 of the derivative's typical size |grad| |d| / sqrt(n)
    times sqrt(n), taken as 1 % of the sum of the absolute products' norm."""
    from speech_amd import ops
    args, go, gs = delta_inputs(75, 2, 2, 2, 16, 24, torch.float32, 6)
    dev = [t.to(cuda) for t in args]
    go, gs = go.to(cuda), gs.to(cuda)

    def loss(xs):
        o, f = ops.gated_delta_rule(*xs[:5], state=xs[5], normalize=True)
        return (o.double() * go).sum() + (f.double() * gs).sum()
    leaves = [t.clone().requires_grad_(True) for t in dev]
    o, f = ops.gated_delta_rule(*leaves[:5], state=leaves[5], normalize=True)
    grads = torch.autograd.grad([o, f], leaves, [go, gs])
    h = 2.0 ** -6
    for i, gr in enumerate(grads):
        d = torch.randn(gr.shape, generator=torch.Generator().manual_seed(i)).to(cuda) * (0.2 if i in (3, 4) else 1.0)
        with torch.no_grad():
            num = (loss([t + h * d if j == i else t for j, t in enumerate(dev)]) - loss([t - h * d if j == i else t for j, t in enumerate(dev)])) / (2 * h)
        ana = (gr.double() * d.double()).sum()
        assert abs(float(num - ana)) <= 0.01 * float((gr.double() * d.double()).norm()), i


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_delta_views(cuda, dtype):
    """q, k, v cut out of one projection (strided views), misaligned and transposed ones, expanded gradients: the same numbers."""
    from speech_amd import ops
    T, B, H, dk, dv = 70, 3, 2, 16, 24
    u = torch.randn(T, B, H * (2 * dk + dv) + 8, device=cuda).to(dtype)
    q, k = u[..., :H * dk].unflatten(-1, (H, dk)), u[..., H * dk:2 * H * dk].unflatten(-1, (H, dk))
    v = u[..., 2 * H * dk:2 * H * dk + H * dv].unflatten(-1, (H, dv))
    g, beta = -torch.rand(B, T, H, device=cuda).transpose(0, 1), torch.rand(T, H, B, device=cuda).transpose(1, 2)
    dense = [t.contiguous() for t in (q, k, v, g, beta)]
    for a in ((q, k, v, g, beta), (q.permute(0, 1, 2, 3), k, v.clone().transpose(0, 1).contiguous().transpose(0, 1), g, beta)):
        for x, y in zip(ops.gated_delta_rule(*a, normalize=True), ops.gated_delta_rule(*dense, normalize=True)):
            assert torch.equal(x, y)
    odd = torch.randn(T * B * H * dk + 1, device=cuda).to(dtype)[1:].view(T, B, H, dk)
    assert torch.equal(ops.gated_delta_rule(odd, k, v, g, beta, normalize=True)[0], ops.gated_delta_rule(odd.clone(), *dense[1:], normalize=True)[0])
    s = torch.randn(B, H, dk, dv, device=cuda)
    so = torch.randn(B * H * dk * dv + 1, device=cuda)[1:].view(B, H, dk, dv)
    so.copy_(s)
    assert torch.equal(ops.gated_delta_rule(*dense, state=so)[1], ops.gated_delta_rule(*dense, state=s)[1])
    leaves = [t.clone().requires_grad_(True) for t in dense]
    o, f = ops.gated_delta_rule(*leaves, normalize=True)
    one = torch.autograd.grad(o.float().sum(), leaves, retain_graph=True)             # an expanded gradient; no gradient of the state
    two = torch.autograd.grad([o, f], leaves, [torch.ones_like(o), torch.zeros_like(f)])
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    leaves = [t.clone().requires_grad_(True) for t in dense]
    o, f = ops.gated_delta_rule(*leaves, normalize=True)
    three = torch.autograd.grad(f.sum(), leaves)                                       # the state's gradient alone: nothing reaches q
    assert not three[0].any() and all(torch.isfinite(t).all() for t in three)
    # one leaf only
    k1 = dense[1].clone().requires_grad_(True)
    ops.gated_delta_rule(dense[0], k1, *dense[2:], normalize=True)[0].float().sum().backward()
    assert torch.equal(k1.grad, one[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("B,Hk,r,dk,dv", [(1, 1, 1, 8, 8), (3, 2, 2, 64, 128), (5, 1, 3, 128, 40)])
def test_delta_step(cuda, dtype, B, Hk, r, dk, dv):
    """Frames one at a time, the state updated in place, are the sequence's."""
    from speech_amd import ops
    args, _, _ = delta_inputs(6, B, Hk, r, dk, dv, dtype, 7)
    dev = [t.to(cuda) for t in args]
    state = dev[5].clone()
    at = state.data_ptr()
    out = torch.stack([ops.gated_delta_step(*(x[t] for x in dev[:5]), state, normalize=True) for t in range(6)])
    ref = [t.double() for t in args]
    ro, rf = delta_reference(*ref, None, dk ** -0.5, True, False)
    assert state.data_ptr() == at
    assert float((state.double().cpu() - rf).norm() / rf.norm()) <= 64 * 2.0 ** -24
    close(out, ro, float(ro.abs().max()), 64 * 6)


def test_delta_step_tells_autograd_of_the_new_state(cuda):
    from speech_amd import ops
    args, _, _ = delta_inputs(1, 2, 2, 1, 16, 16, torch.float32, 7)
    q, k, v, g, beta, state = (t.to(cuda) for t in args)
    w = torch.ones_like(state, requires_grad=True)
    loss = (w * state).sum()                                 # saves the state
    ops.gated_delta_step(q[0], k[0], v[0], g[0], beta[0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        s = state.clone()
        a = ops.gated_delta_step(q[0], k[0], v[0], g[0], beta[0], s)
    b = ops.gated_delta_step(q[0], k[0], v[0], g[0], beta[0], state)
    assert torch.equal(a, b) and torch.equal(s, state)
    o = ops.gated_delta_step(q[0].requires_grad_(True), k[0], v[0], g[0].requires_grad_(True), beta[0], state)
    assert not o.requires_grad and not state.requires_grad


def test_delta_refuses(cuda):
    from speech_amd import ops
    q, v, g = torch.zeros(4, 2, 2, 16, device=cuda), torch.zeros(4, 2, 4, 24, device=cuda), torch.zeros(4, 2, 4, device=cuda)
    s = torch.zeros(2, 4, 16, 24, device=cuda)
    for kw, text in [(dict(k=q[:3]), "must be"), (dict(k=q.half()), "one dtype"), (dict(v=v[:, :, :3]), "evenly"), (dict(g=g[..., :2]), "g and beta"),
                     (dict(beta=g.long()), "g and beta"), (dict(state=s.half()), "state"), (dict(state=s[:1]), "state"), (dict(scale=0.0), "scale"),
                     (dict(scale=float("nan")), "scale"), (dict(lengths=torch.ones(3, dtype=torch.int32, device=cuda)), "lengths"),
                     (dict(lengths=torch.ones(2, device=cuda)), "lengths"), (dict(lengths=torch.ones(2, dtype=torch.int32)), "lengths is on"),
                     (dict(lengths=torch.ones(2, dtype=torch.bool, device=cuda)), "lengths"),
                     (dict(q=torch.zeros(4, 2, 2, 12, device=cuda), k=torch.zeros(4, 2, 2, 12, device=cuda)), "multiples of 8"),
                     (dict(q=q[:, :, :1], k=q[:, :, :1], bidirectional=True), "even"), (dict(state=s.cpu()), "state is on")]:
        a = dict(q=q, k=q, v=v, g=g, beta=g)
        a.update(kw)
        with pytest.raises(ValueError, match=text):
            ops.gated_delta_rule(**a)
    for st, text in ((None, "state"), (s.transpose(2, 3).contiguous().transpose(2, 3), "contiguous"), (s.clone().requires_grad_(True), "differentiable")):
        with pytest.raises(ValueError, match=text):
            ops.gated_delta_step(q[0], q[0], v[0], g[0], g[0], st)
    leaf = q.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(ops.gated_delta_rule(leaf, q, v, g, g)[0].sum(), leaf, create_graph=True)
    # nothing to do
    o, f = ops.gated_delta_rule(q[:0], q[:0], v[:0], g[:0], g[:0], state=s + 1)
    assert o.shape == (0, 2, 4, 24) and torch.equal(f, s + 1)
    o, f = ops.gated_delta_rule(q[:, :0], q[:, :0], v[:, :0], g[:, :0], g[:, :0])
    assert o.shape == (4, 0, 4, 24) and f.shape == (0, 4, 16, 24)


def test_delta_repeats_bit_for_bit(cuda):
    from speech_amd import ops
    args, go, gs = delta_inputs(200, 6, 4, 2, 64, 128, torch.bfloat16, 8)
    first = None
    for _ in range(3):
        xs = [t.to(cuda).requires_grad_(True) for t in args]
        o, f = ops.gated_delta_rule(*xs[:5], state=xs[5], normalize=True, bidirectional=True)
        out = [o.detach(), f.detach(), *torch.autograd.grad([o, f], xs, [go.to(cuda), gs.to(cuda)])]
        first = first or out
        assert all(torch.equal(u, v) for u, v in zip(out, first))


def test_delta_strides_of_size_one_and_far_frames(cuda):
    """A dimension of size one may carry any stride; frames may lie far apart: the same numbers as from dense tensors."""
    from speech_amd import ops
    base = torch.randn(4000, device=cuda)
    q, k = (base.as_strided((1, 1, 2, 16), (33, 35, 16, 1), o) for o in (0, 40))
    v = base.as_strided((1, 1, 2, 24), (7, 5, 24, 1), 100)
    g, beta = -torch.rand(1, 1, 2, device=cuda), torch.rand(1, 1, 2, device=cuda)
    for train in (False, True):
        a = [t.detach().requires_grad_(train) for t in (q, k, v, g, beta)]
        b = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(train) for t in (q, k, v, g, beta)]
        (o, f), (p, e) = ops.gated_delta_rule(*a, normalize=True), ops.gated_delta_rule(*b, normalize=True)
        assert torch.equal(o, p) and torch.equal(f, e)
        if train:
            assert all(torch.equal(x, y) for x, y in zip(torch.autograd.grad(o.sum(), a), torch.autograd.grad(p.sum(), b)))
    far = torch.zeros(20, (1 << 23) + 8, device=cuda)
    q = far[:, :32].view(20, 1, 2, 16)
    q.copy_(torch.randn(20, 1, 2, 16, device=cuda))
    v, g, beta = torch.randn(20, 1, 2, 24, device=cuda), -torch.rand(20, 1, 2, device=cuda), torch.rand(20, 1, 2, device=cuda)
    for n in (20, 5):
        x = ops.gated_delta_rule(q[:n], q[:n], v[:n], g[:n], beta[:n], normalize=True)
        y = ops.gated_delta_rule(q[:n].clone(), q[:n].clone(), v[:n], g[:n], beta[:n], normalize=True)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_group_norm_without_frames(cuda):
    from speech_amd import ops
    x = torch.zeros(2, 0, 8, device=cuda, requires_grad=True)
    w, b = torch.ones(8, device=cuda, requires_grad=True), torch.zeros(8, device=cuda, requires_grad=True)
    y = ops.group_norm(x, w, b, 2, act="silu")
    gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
    assert y.shape == x.shape == gx.shape and not gw.any() and not gb.any()
    one = torch.randn(3, 1, 1, 8, device=cuda).as_strided((3, 1, 1, 8), (8, 3, 5, 1))
    assert torch.equal(ops.group_norm(one, w, b, 2), ops.group_norm(one.clone(memory_format=torch.contiguous_format), w, b, 2))


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_delta_step_takes_any_view(cuda, dtype):
    """Odd first elements, odd strides, gates with gaps: the numbers of dense tensors."""
    from speech_amd import ops
    base = torch.randn(9000, device=cuda).to(dtype)
    q, k = (base.as_strided((3, 2, 24), (1001, 31, 1), o) for o in (1, 501))
    v = base.as_strided((3, 4, 40), (2003, 83, 1), 4003)
    g, beta = -torch.rand(3, 9, device=cuda)[:, 1::2], torch.rand(4, 3, device=cuda).t()
    state = torch.randn(3, 4, 24, 40, device=cuda)
    other = state.clone()
    o = ops.gated_delta_step(q, k, v, g, beta, state, normalize=True)
    dense = [t.clone(memory_format=torch.contiguous_format) for t in (q, k, v, g, beta)]
    assert torch.equal(o, ops.gated_delta_step(*dense, other, normalize=True)) and torch.equal(state, other)
    rule = ops.gated_delta_rule(*(t[None] for t in (q, k, v, g, beta)), state=torch.randn(3, 4, 24, 40, device=cuda) * 0 + other, normalize=True)
    assert torch.equal(rule[0][0], ops.gated_delta_step(*dense, other, normalize=True)) and torch.equal(rule[1], other)


@pytest.mark.parametrize("T", [7, 100])
def test_in_place_entry_points(cuda, T):
    """The C ABI's in-place forms: state_out = state of both forward forms, y = x and y = residual of the dropout."""
    from speech_amd import _lib, ops
    h = _lib.lib()
    args, _, _ = delta_inputs(T, 2, 2, 2, 16, 40, torch.bfloat16, 3)
    q, k, v, g, beta, state = (t.to(cuda) for t in args)
    o, final = ops.gated_delta_rule(q, k, v, g, beta, state=state)
    o2 = torch.empty_like(o)
    n = h.sp_gdr_workspace_bytes(T, 2, 2, 4, 16, 40, _lib.SP_BF16, 0)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    strides = ops._strides(q, k, v, g, beta)
    _lib.check(h.sp_gdr_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(), None, strides, T, 2, 2, 4, 16, 40,
                            16 ** -0.5, 0, _lib.SP_BF16, o2.data_ptr(), state.data_ptr(), None, 0, ws.data_ptr(), n, ops.raw_stream(q)))
    assert torch.equal(o, o2) and torch.equal(final, state)
    x, r = torch.randn(1003, device=cuda), torch.randn(1003, device=cuda)
    rng = ops.dropout_rng(4, cuda)
    want = ops.dropout(x, 0.3, rng, 1, residual=r)
    for y in (x.clone(), r.clone()):
        a, b = (y, r) if torch.equal(y, x) else (x, y)
        _lib.check(h.sp_dropout(a.data_ptr(), b.data_ptr(), 1, 1003, 0.3, rng.data_ptr(), 1, _lib.SP_F32, y.data_ptr(), None, ops.raw_stream(x)))
        assert torch.equal(y, want)


def test_offsets_beyond_32_bits(cuda):
    """Samples, utterances and elements that lie more than 2^32 bytes and 2^31 elements into a tensor."""
    from speech_amd import ops
    far = (1 << 31) + 4096
    base = torch.empty(far + (1 << 16), dtype=torch.bfloat16, device=cuda)
    x = base.as_strided((2, 3, 10, 32), (far, 320, 32, 1))
    x.copy_(torch.randn(2, 3, 10, 32, device=cuda))
    w, b = torch.rand(32, device=cuda), torch.rand(32, device=cuda)
    dense = x.clone(memory_format=torch.contiguous_format)
    assert torch.equal(ops.group_norm(x, w, b, 4, act="silu", residual=x), ops.group_norm(dense, w, b, 4, act="silu", residual=dense))
    xg, dg = x.detach().requires_grad_(True), dense.requires_grad_(True)
    assert torch.equal(torch.autograd.grad(ops.group_norm(xg, w, b, 4).float().square().sum(), xg)[0],
                       torch.autograd.grad(ops.group_norm(dg, w, b, 4).float().square().sum(), dg)[0])
    for T in (3, 70):
        q = base.as_strided((T, 2, 2, 16), (32, far, 16, 1))
        q.copy_(torch.randn(T, 2, 2, 16, device=cuda))
        g = -torch.rand(T, 2, 2, device=cuda)
        a = ops.gated_delta_rule(q, q, q, g, -g, normalize=True)
        d = q.clone(memory_format=torch.contiguous_format)
        c = ops.gated_delta_rule(d, d, d, g, -g, normalize=True)
        assert torch.equal(a[0], c[0]) and torch.equal(a[1], c[1])
    base.fill_(1.0)
    y = ops.dropout(base, 0.5, ops.dropout_rng(6, cuda, 2), 1)
    u = np.uint64
    at = np.arange((base.numel() - 4096) // 8, base.numel() // 8, dtype=u)
    c = [at & u(0xFFFFFFFF), at >> u(32), np.full_like(at, 2), np.full_like(at, 1)]
    for r in range(10):
        p0, p1 = u(0xD2511F53) * c[0], u(0xCD9E8D57) * c[2]
        c = [(p1 >> u(32)) ^ c[1] ^ u((6 + r * 0x9E3779B9) & 0xFFFFFFFF), p1 & u(0xFFFFFFFF), (p0 >> u(32)) ^ c[3] ^ u((r * 0xBB67AE85) & 0xFFFFFFFF), p0 & u(0xFFFFFFFF)]
    keep = np.stack(c, -1).astype("<u4").view("<u2").reshape(-1) >= 32768
    assert torch.equal(y[-4096:].cpu() != 0, torch.from_numpy(keep))


# ------------------------------------------------------------------------------------------ streams, graphs, the operators together
def _layer(cuda, dtype=torch.bfloat16):
    from speech_amd import net
    torch.manual_seed(3)
    layer = net.GatedDeltaLayer(64, 64, heads=4, dk=16, dropout=0.2, site=2).to(cuda)
    with torch.no_grad():
        layer.group_norm.weight.uniform_(0.5, 1.5)
        layer.layer_norm.bias.uniform_(-0.2, 0.2)
    return layer, torch.randn(70, 3, 64, device=cuda).to(dtype)


def test_other_stream(cuda):
    """Everything is enqueued on the caller's stream."""
    from speech_amd import ops
    layer, x = _layer(cuda)
    rng = ops.dropout_rng(5, cuda)
    want = layer(x, rng)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        big = torch.randn(4096, 4096, device=cuda)
        for _ in range(20):
            big = big @ big * 1e-3
        late = torch.where(big.sum() == 123.456, torch.zeros_like(x), x)          # ready only behind the products
        got = layer(late, rng)[0]
        total = got.float().sum()
    s.synchronize()
    assert torch.equal(got, want) and torch.isfinite(total)


def test_layer_against_plain_torch(cuda):
    """The run of operators of an encoder layer (projection -> delta rule -> group norm with SiLU -> projection -> dropout + residual), forward
    and gradients, against the same layer stated in f64.  f32 activations: the products run on the f32 matrix instruction, so every step is
    within a few f32 roundings; 2^-24 * 2048 of the two-norm covers the chain of six."""
    from speech_amd import ops
    layer, x = _layer(cuda, torch.float32)
    rng = ops.dropout_rng(11, cuda, 4)
    lengths = torch.tensor([70, 31, 0], device=cuda)
    x = x.requires_grad_(True)
    y, final = layer(x, rng, lengths)
    gy = torch.randn(y.shape, generator=torch.Generator().manual_seed(1)).to(cuda)
    names, params = zip(*layer.named_parameters())
    got = torch.autograd.grad(y, [x, *params], gy)
    P = {n: p.detach().double().cpu().requires_grad_(True) for n, p in layer.named_parameters()}
    x64 = x.detach().double().cpu().requires_grad_(True)
    H, dk, dv = 4, 16, 16
    u = torch.nn.functional.layer_norm(x64, (64,), P["layer_norm.weight"], P["layer_norm.bias"]) @ P["w_in"]
    q, k, v = (u[..., a:a + n].unflatten(-1, (H, -1)) for a, n in ((0, 64), (64, 64), (128, 64)))
    g = -torch.exp(P["a_log"]) * torch.nn.functional.softplus(u[..., 192:196] + P["a_bias"])
    o, rf = delta_reference(q, k, v, g, torch.sigmoid(u[..., 196:200]), None, [70, 31, 0], dk ** -0.5, True, True)
    z = torch.nn.functional.group_norm(o.reshape(-1, 64), H, P["group_norm.weight"], P["group_norm.bias"], 1e-5)
    z = (z * torch.sigmoid(z)) @ P["w_out"]
    thr = round(0.2 * 65536)
    keep = (philox_draws(x.numel(), 11, 4, 2) >= thr).view(x.shape)
    ref = torch.where(keep, z.view(x.shape) * (65536 / (65536 - thr)), 0.0) + x64
    want = torch.autograd.grad(ref, [x64, *(P[n] for n in names)], gy.double().cpu())
    for name, u_, w_ in [("y", y, ref), ("final", final, rf)] + list(zip(("x", *names), got, want)):
        e = float((u_.detach().double().cpu() - w_.detach()).norm() / w_.detach().norm())
        assert e <= 2048 * 2.0 ** -24, (name, e)


def test_stack_is_not_twice_differentiable(cuda):
    from speech_amd import net
    m = net.SRModel(1, 64, 28, 80, 0.0, norm="group", rnn="delta").to(cuda).train()
    loss = m(torch.rand(1, 1, 80, 20, device=cuda)).sum()
    for p in (m.cnn.weight, m.resnet_layers[0].conv1.weight):
        with pytest.raises(RuntimeError, match="twice"):
            torch.autograd.grad(loss, p, create_graph=True)


def test_graph_capture(cuda):
    """A training pass of the layer captured once and replayed, with eager work between: the dropout follows the generator state, which the
    graph advances itself; every replay equals the eager pass of that step."""
    from speech_amd import ops
    layer, x0 = _layer(cuda)
    x = x0.clone().requires_grad_(True)
    gy = torch.randn_like(x0)
    rng = ops.dropout_rng(21, cuda)
    leaves = [x, *layer.parameters()]

    def step():
        y, _ = layer(x, rng)
        return [y, *torch.autograd.grad(y, leaves, gy)]

    def eager(xv, at):
        with torch.no_grad():
            xl = xv.clone()
        xl.requires_grad_(True)
        y, _ = layer(xl, ops.dropout_rng(21, cuda, at))
        return [y.detach(), *torch.autograd.grad(y, [xl, *layer.parameters()], gy)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [t.detach() for t in step()]
        rng[1] += 1
    for at in range(4):
        xv = torch.randn(x0.shape, generator=torch.Generator().manual_seed(at)).to(cuda).to(x0.dtype)
        want = eager(xv, at)
        with torch.no_grad():
            x.copy_(xv)
        graph.replay()
        torch.cuda.synchronize()
        assert int(rng[1]) == at + 1
        for i, u, w in zip(("y", "x", *(n for n, _ in layer.named_parameters())), out, want):
            # the layer norm's parameter gradients are summed with float atomics (two half f32 steps a block of 70 * 3 rows), all else bit for bit
            if i.startswith("layer_norm"):
                assert torch.allclose(u, w, rtol=0, atol=256 * 2.0 ** -24 * float(w.abs().max())), i
            else:
                assert torch.equal(u, w), i
    # two graphs with workspaces of their own, replayed in turn
    g2 = torch.cuda.CUDAGraph()
    x2 = torch.randn_like(x0)
    with torch.no_grad(), torch.cuda.graph(g2):
        o2 = ops.group_norm(x2, layer.group_norm.weight, layer.group_norm.bias, 4, act="silu")
    with torch.no_grad():
        w2 = ops.group_norm(x2, layer.group_norm.weight, layer.group_norm.bias, 4, act="silu")
    for _ in range(3):
        graph.replay()
        g2.replay()
        torch.cuda.synchronize()
        assert torch.equal(o2, w2)


def test_layer_streams_frame_by_frame(cuda):
    """GatedDeltaLayer.step over the frames is the unidirectional layer over the sequence."""
    from speech_amd import net
    torch.manual_seed(5)
    layer = net.GatedDeltaLayer(64, 64, heads=4, dk=16, bidirectional=False).to(cuda).eval()
    x = torch.randn(40, 2, 64, device=cuda)
    with torch.no_grad():
        want, final = layer(x)
    state = torch.zeros(2, 4, 16, 16, device=cuda)
    got = torch.stack([layer.step(x[t], state) for t in range(40)])
    assert float((got - want).norm() / want.norm()) <= 2048 * 2.0 ** -24
    assert float((state - final).norm() / final.norm()) <= 2048 * 2.0 ** -24
    with pytest.raises(RuntimeError, match="frame by frame"):
        net.GatedDeltaLayer(64, 64, heads=4, dk=16).to(cuda).step(x[0], state)


@pytest.mark.parametrize("norm,rnn", [("group", "sru"), ("batch", "delta"), ("group", "delta")])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=ids)
def test_model_variants_train_and_evaluate(cuda, norm, rnn, dtype):
    """A training step through train.train_step changes every parameter, evaluation runs, a checkpoint round trip gives the same logits."""
    from speech_amd import net
    from speech_amd.train import FlatAdam, train_step
    torch.manual_seed(2)
    m = net.SRModel(2, 64, 28, 80, 0.1, compute_dtype=dtype, norm=norm, rnn=rnn).to(cuda).train()
    with torch.no_grad():
        for blk in m.resnet_layers:
            blk.bn2.weight.fill_(0.5)
    opt = FlatAdam(m.parameters(), lr=1e-2)
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    spec = torch.rand(3, 1, 80, 61, device=cuda)
    labels = torch.randint(1, 29, (3, 6), device=cuda)
    ll = torch.tensor([6, 4, 5], dtype=torch.int32, device=cuda)
    for _ in range(2):
        assert torch.isfinite(train_step(m, opt, spec, labels, ll))
    for n, p in m.named_parameters():
        if norm == "batch" and "conv" in n and n.endswith("bias"):
            continue            # a bias in front of batch statistics has no gradient
        assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n
    if rnn == "delta":
        assert int(m.delta_layers.dropout_state[1]) == 2
    m.eval()
    with torch.no_grad():
        a = m(spec)
        other = net.SRModel(2, 64, 28, 80, 0.1, compute_dtype=dtype, norm=norm, rnn=rnn).to(cuda).eval()
        other.load_checkpoint(m.state_dict())
        assert torch.isfinite(a).all() and torch.equal(a, other(spec))
        if norm == "group":      # no utterance sees another
            assert torch.equal(m(spec[:1]), a[:1]) or float((m(spec[:1]) - a[:1]).abs().max()) <= 1e-2 * float(a.abs().max())


class _Bf16(torch.autograd.Function):
    """Rounds a value on the way forward and its gradient on the way back, as a bf16 tensor between two kernels does."""

    @staticmethod
    def forward(ctx, x):
        return x.to(torch.bfloat16).double()

    @staticmethod
    def backward(ctx, g):
        return g.to(torch.bfloat16).double()


class _Bf16Weight(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        return x.to(torch.bfloat16).double()

    @staticmethod
    def backward(ctx, g):
        return g


def _group_stack_reference(m, spec, rnd, rw):
    """cnn and blocks of a model in f64 with `rnd` at every activation that the bf16 stack writes and `rw` at the 3 x 5 weights."""
    x = rnd(m.cnn(spec))
    for blk in m.resnet_layers:
        conv = lambda t, c: rnd(torch.nn.functional.conv2d(t, rw(c.weight), None, 1, c.padding))      # noqa: E731
        y = rnd(torch.relu(blk.bn1(conv(x, blk.conv1))))
        x = rnd(torch.relu(blk.bn2(conv(y, blk.conv2)) + x))
    return x.permute(3, 0, 2, 1).reshape(x.shape[3], x.shape[0], -1)


def test_group_conv_stack_against_plain_torch(cuda):
    """The conv stack with group norm.  f32 evaluation: against the plain f64 statement within f32 rounding (seven convolutions of up to 480
    products, 2^-24 * 4096 of the two-norm).  The bf16 stack: against the f64 statement that rounds at the same places.

    Where an f32 sum rounds the other way the two differ by one bf16 step.  A convolution spreads such a difference d (relative) over its
    neighbours, and rounding to steps of 2^-8 turns d into whole steps with probability d / 2^-8: an rms of sqrt(d 2^-8), more than d.  From
    2^-12 in the first activation that is 2^-10, 2^-9, ..., so after a few layers the two sides differ by up to an rms of 2^-8 of the values,
    however exact the kernels are: the forward bound is twice that, 2^-7.  On the way back each of the six ReLUs stops or passes a whole
    gradient where its argument (density at zero <= 0.4 per standard deviation) lies within that difference (mean size 0.8 * 2^-8): a
    fraction 0.4 * 0.8 * 2^-8 = 2^-9.6 of the elements, 2^-4.8 of the two-norm, for six of them 2^-4.8 * sqrt(6) = 2^-3.5 = 0.088.  The
    roundings of 13 gradients (sqrt(13) 2^-9) vanish in that.  The bound shows that the stack is put together rightly; the precision of its
    steps is the other tests' matter."""
    from speech_amd import convstack, net
    torch.manual_seed(4)
    m = net.SRModel(1, 64, 28, 80, 0.0, norm="group").to(cuda)
    with torch.no_grad():
        for blk in m.resnet_layers:
            blk.bn2.weight.uniform_(0.5, 1.0)
            blk.bn1.bias.uniform_(-0.3, 0.3)
    spec = torch.rand(2, 1, 80, 75, device=cuda)
    P = net.SRModel(1, 64, 28, 80, 0.0, norm="group").double()
    P.load_state_dict({k: v.cpu() for k, v in m.state_dict().items()})
    same = lambda t: t      # noqa: E731
    rel = lambda u, w: float((u.detach().double().cpu() - w.detach()).norm() / w.detach().norm())      # noqa: E731
    with torch.no_grad():
        f32 = convstack.conv_stack_group(spec, m.cnn, list(m.resnet_layers), True)
        want = _group_stack_reference(P, spec.double().cpu(), same, same)
    assert f32.dtype == torch.float32 and rel(f32, want) <= 4096 * 2.0 ** -24, rel(f32, want)
    out = convstack.conv_stack_group(spec, m.cnn, list(m.resnet_layers))
    ref = _group_stack_reference(P, spec.double().cpu(), _Bf16.apply, _Bf16Weight.apply)
    assert out.dtype == torch.bfloat16 and rel(out, ref) <= 2.0 ** -7, rel(out, ref)
    gy = torch.randn(out.shape, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    names, params = zip(*[(n, p) for n, p in m.named_parameters() if n.startswith(("cnn", "resnet_layers"))])
    got = torch.autograd.grad(out, params, gy.to(cuda))
    grads = torch.autograd.grad(ref, [dict(P.named_parameters())[n] for n in names], gy.double())
    errors = {n: rel(u, w) for n, u, w in zip(names, got, grads)}
    assert max(errors.values()) <= 0.088, errors


def test_conv_functions_of_the_group_stack(cuda):
    """The two convolutions that the stack differentiates by themselves, against f64 on the values they are given (bf16 activations; 3 x 5
    weights are rounded to bf16, which the reference repeats).  y and gx: a half step of the value and f32 sums of at most 480 products (depth
    480); parameter gradients: f32 sums over all positions, here 2 * 10 * 37 products each."""
    from speech_amd import convstack
    torch.manual_seed(6)
    x, w = torch.randn(2, 10, 37, 32).to(torch.bfloat16), (torch.randn(32, 32, 3, 5) / 20).to(torch.bfloat16).float()
    gy = torch.randn(2, 10, 37, 32).to(torch.bfloat16)
    xd, wd = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    y = convstack._Conv3x5Fn.apply(xd, wd)
    gx, gw = torch.autograd.grad(y, [xd, wd], gy.to(cuda))
    x64, w64 = x.double().requires_grad_(True), w.double().requires_grad_(True)
    ref = torch.nn.functional.conv2d(x64.permute(0, 3, 1, 2), w64, None, 1, (1, 2)).permute(0, 2, 3, 1)
    rx, rw = torch.autograd.grad(ref, [x64, w64], gy.double())
    close(y, ref, float(ref.detach().abs().max()), 480)
    close(gx, rx, float(rx.abs().max()), 480)
    close(gw, rw, float(rw.abs().max()), 740, torch.float32)
    spec, ws, bs = torch.rand(2, 1, 21, 75), torch.randn(32, 1, 3, 3), torch.randn(32)
    leaves = [t.to(cuda).requires_grad_(True) for t in (ws, bs)]
    y = convstack._StemFn.apply(spec.to(cuda), *leaves)
    gy = torch.randn(y.shape).to(torch.bfloat16)
    r = [t.double().requires_grad_(True) for t in (ws, bs)]
    ref = torch.nn.functional.conv2d(spec.double(), *r, 2, 1).permute(0, 2, 3, 1)
    close(y, ref, float(ref.detach().abs().max()), 16)
    for u, v in zip(torch.autograd.grad(y, leaves, gy.to(cuda)), torch.autograd.grad(ref, r, gy.double())):
        close(u, v, float(v.abs().max()), 836, torch.float32)


def test_concurrent_streams(cuda):
    """Two streams run training passes of the layer at the same time: no workspace is shared, each gets the results of a run alone."""
    from speech_amd import ops
    layer, x = _layer(cuda)
    gy = torch.randn_like(x)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    inputs = [x, torch.randn_like(x)]

    def run(xv, seed):
        xl = xv.clone().requires_grad_(True)
        y, f = layer(xl, ops.dropout_rng(seed, cuda))
        return [y.detach(), f.detach(), torch.autograd.grad(y, xl, gy)[0]]
    want = [run(v, i) for i, v in enumerate(inputs)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(inputs[i], i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert all(torch.equal(u, w) for u, w in zip(g, want[i]))


def test_variant_trains_resumes_and_evaluates_from_the_commands(cuda, tmp_path, monkeypatch):
    """`--norm group --rnn delta` through train.main (synthetic clips), its checkpoint through --resume and through
    scripts/eval_dataset's model construction."""
    import wave
    from speech_amd import train
    from speech_amd.scripts import eval_dataset as ev
    monkeypatch.delenv("WORLD_SIZE", raising=False)
    ckpt = tmp_path / "variant.pth"
    args = ["--one_iter", "--synthetic", "--synthetic_clips", "16", "--steps", "2", "--multiplier", "1", "--num_workers", "0", "--norm", "group",
            "--rnn", "delta", "--dtype", "bf16", "--checkpoint", str(ckpt)]
    hp = train.parse_args(args)
    hp.update(batch_size=4, n_rnn_layers=2, rnn_dim=64)
    assert np.isfinite(train.main(hp))
    hp = train.parse_args(args + ["--resume", str(ckpt)])
    hp.update(batch_size=4, n_rnn_layers=2, rnn_dim=64, epochs=2, one_iter=False)
    assert torch.load(ckpt, weights_only=True)["model_state_dict"]["delta_layers.dropout_state"].tolist() == [7, 2]
    assert np.isfinite(train.main(hp))
    ibm = tmp_path / "ibm"
    ibm.mkdir()
    rs = np.random.RandomState(4)
    for k in range(3):
        with wave.open(str(ibm / f"i{k}.wav"), "wb") as f:
            f.setnchannels(1); f.setsampwidth(2); f.setframerate(16000)
            f.writeframes((rs.randn(6000 + 300 * k) * 2500).clip(-32768, 32767).astype("<i2").tobytes())
        (ibm / f"i{k}.txt").write_text("ibm line")
    for dtype in ("fp16", "fp32"):
        cer, _ = ev.main(["False", "ibm", str(ckpt), "--ibm_root", str(ibm), "--n_rnn_layers", "2", "--rnn_dim", "64", "--batch_size", "2",
                          "--num_workers", "0", "--norm", "group", "--rnn", "delta", "--dtype", dtype], log=lambda *a: None)
        assert np.isfinite(cer)
