"""Group normalisation, dropout and the gated delta rule at their edges: precision of 16-bit results, long walks of a thread, the scans' wide
form, padding that must have no influence, calls that must be refused.  References are stated in 64 bits on the CPU."""
import pytest
import torch

from test_gpu_operators import DTYPES, close, delta_inputs, delta_reference, gn_inputs, gn_reference, ids

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


def _gn_compare(cuda, x, w, b, r, gy, G, act, lengths=None, xd=None, rd=None, gyd=None, time_major=False):
    """Values and gradients against the 64-bit statement; xd, rd, gyd: the same tensors on the GPU in another layout."""
    from speech_amd import ops
    xd, rd = ((t if d is None else d) for t, d in ((x.to(cuda), xd), (r.to(cuda) if r is not None else None, rd)))
    gyd = gy.to(cuda) if gyd is None else gyd
    leaves = [t.detach().requires_grad_(True) for t in (xd, w.to(cuda), b.to(cuda), rd) if t is not None]
    L = None if lengths is None else torch.tensor(lengths, device=cuda)
    y = ops.group_norm(*leaves[:3], G, act=act, residual=leaves[3] if rd is not None else None, lengths=L, time_major=time_major)
    ref = [t.double().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    ry = gn_reference(*ref[:3], G, act, ref[3] if r is not None else None, lengths)
    got, want = torch.autograd.grad(y, leaves, gyd), torch.autograd.grad(ry, ref, gy.double())
    scale = float(ry.detach().abs().max()) + 8
    # chains: a thread's positions (at most 32 here) four at a time, eight rows of partial results, trees: fewer than 256 roundings
    close(y, ry, scale, 256, what="y")
    terms = float(gy.abs().max() * w.abs().max()) * 6 * 2       # rstd is below 2 for these inputs (spread 1.5)
    close(got[0], want[0], terms, 512, what="dx")
    m = x[..., 0].numel()
    for k in (1, 2):      # sums of m terms of size <= 8 gy, in chains of 32 positions, 96 rows a chain behind them and trees
        close(got[k], want[k], float(gy.abs().max()) * 8 * m ** 0.5 + float(want[k].abs().max()), 512, torch.float32, "parameters")
    if rd is not None:
        close(got[3], want[3], float(gy.abs().max()) * 2, 64, what="dres")
    return y, got


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("layout", ["dense", "gaps", "time_major"])
def test_group_norm_long_walks(cuda, dtype, ragged, layout):
    """150 samples of 7 bands of 101 frames, 64 channels: splits of 142 positions, 32 rows of threads, four and a half positions a thread; a walk
    crosses the ends of bands.  gaps: bands and frames with memory between them; time_major: gradients arrive in the order that the result was
    written in."""
    x, w, b, r, gy = gn_inputs((150, 7, 101, 64), dtype, 4, True)
    lengths = [101 - (n * 37) % 102 if n % 2 else 101 for n in range(150)] if ragged else None
    kw = {}
    if layout == "gaps":
        def spread(t):
            base = torch.full((150, 9, 104, 80), float("nan"), dtype=dtype, device=cuda)
            base[:, 1:8, 2:103, 8:72] = t.to(cuda)
            return base[:, 1:8, 2:103, 8:72]
        kw = dict(xd=spread(x), rd=spread(r), gyd=spread(gy))
    elif layout == "time_major":
        kw = dict(time_major=True, gyd=gy.to(cuda).permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3))
    y, got = _gn_compare(cuda, x, w, b, r, gy, 8, "silu", lengths, **kw)
    if layout == "time_major":
        assert y.permute(2, 0, 1, 3).is_contiguous()
    if ragged:
        for n, v in enumerate(lengths):
            assert not y[n, :, v:].any() and not got[0][n, :, v:].any() and not got[3][n, :, v:].any()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("res,act", [(True, "silu"), (False, "none")])
def test_group_norm_rows_in_turn(cuda, dtype, res, act):
    """40000 samples of one position, 256 channels in 8 groups: a team of lanes takes two or three units forwards and six or seven backwards,
    each one's loads ahead of the one before, the parameters' gradients summed in registers on the way."""
    x, w, b, r, gy = gn_inputs((40000, 1, 1, 256), dtype, 5, res)
    _gn_compare_rows(cuda, x, w, b, r, gy, 8, act)


def _gn_compare_rows(cuda, x, w, b, r, gy, G, act):
    from speech_amd import ops
    leaves = [t.to(cuda).requires_grad_(True) for t in (x, w, b, r) if t is not None]
    y = ops.group_norm(*leaves[:3], G, act=act, residual=leaves[3] if r is not None else None)
    ref = [t.double().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    v = ref[0].unflatten(-1, (G, -1))
    m = v.mean(-1, keepdim=True)
    z = ((v - m) / torch.sqrt(((v - m) ** 2).mean(-1, keepdim=True) + 1e-5)).flatten(-2) * ref[1] + ref[2]
    z = z + ref[3] if r is not None else z
    ry = z * torch.sigmoid(z) if act == "silu" else z
    got, want = torch.autograd.grad(y, leaves, gy.to(cuda)), torch.autograd.grad(ry, ref, gy.double())
    close(y, ry, float(ry.detach().abs().max()) + 8, 128, what="y")
    rstd = float((1 / torch.sqrt(v.detach().var(-1, unbiased=False) + 1e-5)).max())
    close(got[0], want[0], rstd * float(gy.abs().max() * w.abs().max()) * 6, 256, what="dx")
    for k in (1, 2):
        close(got[k], want[k], float(gy.abs().max()) * 8 * x.shape[0] ** 0.5 + float(want[k].abs().max()), 512, torch.float32, "parameters")
    if r is not None:
        close(got[3], want[3], float(gy.abs().max()) * 2, 64, what="dres")


@pytest.mark.parametrize("shape", [(2, 1, 40, 2048, 1), (2, 2, 20, 2040, 3), (3, 1, 33, 1026, 2)], ids=str)
@pytest.mark.parametrize("offset", [2, 4])
@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
def test_group_norm_several_passes_of_channels(cuda, dtype, shape, offset):
    """Tensors aligned to two or four elements only: more chunks of channels than a workgroup has threads, and groups that lie in two passes."""
    *s, G = shape
    x, w, b, r, gy = gn_inputs(s, dtype, 6, True)

    def shift(t):
        base = torch.empty(t.numel() + 8, dtype=dtype, device=cuda)
        v = base[offset:offset + t.numel()].view(t.shape)
        v.copy_(t.to(cuda))
        return v
    _gn_compare(cuda, x, w, b, r, gy, G, "silu", None, shift(x), shift(r), shift(gy))


# ------------------------------------------------------------------------------------------ the scans' wide form
def heads_reference(args, lengths, bidirectional, go=None, gs=None):
    """The gated delta rule (q and k normalised) frame by frame in 64 bits, all heads of all utterances at once."""
    q, k, v, g, beta, S = (t.double().requires_grad_(go is not None) for t in args)
    leaves = [q, k, v, g, beta, S]
    T, B, Hk, dk = q.shape
    H = v.shape[2]
    n = torch.tensor(lengths)
    t = torch.arange(T)[:, None]
    back = torch.where(t < n, n - 1 - t, t)                       # [T, B]: an utterance's own frames backwards

    def turn(x):
        if not bidirectional:
            return x
        h = x.shape[2] // 2
        at = back.view(T, B, 1, *[1] * (x.dim() - 3)).expand(T, B, h, *x.shape[3:])
        return torch.cat([x[:, :, :h], torch.gather(x[:, :, h:], 0, at)], 2)
    qh, kh = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    qh, kh = (turn(x).repeat_interleave(H // Hk, 2) for x in (qh * dk ** -0.5, kh))
    vh, gh, bh = turn(v), turn(g), turn(beta)
    out = []
    for i in range(T):
        on = (i < n).view(B, 1, 1)
        s1 = torch.exp(gh[i])[..., None, None] * S
        u = bh[i][..., None] * (vh[i] - (kh[i][..., None] * s1).sum(-2))
        s1 = s1 + kh[i][..., None] * u[..., None, :]
        out.append(torch.where(on, (qh[i][..., None] * s1).sum(-2), 0.0))
        S = torch.where(on[..., None], s1, S)
    o = turn(torch.stack(out))
    if go is None:
        return [o.detach(), S.detach()]
    clean = torch.where((t < n)[..., None, None], go.double(), 0.0)
    return [o.detach(), S.detach(), *torch.autograd.grad([o, S], leaves, [clean, gs.double()])]


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("dk", [64, 72, 128])
@pytest.mark.parametrize("dv", [72, 128])
@pytest.mark.parametrize("train", [False, True])
def test_delta_wide_scans(cuda, dtype, dk, dv, train):
    """More than 128 heads and columns: scans of eight waves.  17 utterances of 8 heads, three chunks, ragged, both directions.  Three utterances
    against the 64-bit statement (bounds as in test_gpu_operators.delta_check, 16-bit results as rounded_once), all of them against the same
    utterances in two calls of the narrow form: the same sums in the same order but for what the compiler joins to a multiply-add, so
    within the same f32 bound, and a 16-bit result within two roundings of it."""
    from speech_amd import ops
    T, B = 150, 17
    args, go, gs = delta_inputs(T, B, 8, 1, dk, dv, dtype, 21, unit=False)
    lengths = [150 - (b * 29) % 151 if b % 3 else 150 for b in range(B)]
    lengths[1], lengths[16] = 0, 129

    def run(sel):
        xs = [(t[sel] if i == 5 else t[:, sel]).to(cuda).requires_grad_(train) for i, t in enumerate(args)]
        o, f = ops.gated_delta_rule(*xs[:5], state=xs[5], lengths=torch.tensor(lengths)[sel].to(cuda), normalize=True, bidirectional=True)
        out = [o, f]
        if train:
            out += torch.autograd.grad([o, f], xs, [go[:, sel].to(cuda), gs[sel].to(cuda)])
        return [t.detach().cpu() for t in out]
    wide = run(slice(0, B))
    halves = [run(slice(0, 8)), run(slice(8, B))]
    which = lambda i: 0 if i in (1, 7) else 1      # noqa: E731      # the batch dimension: states [B, ..], everything else [T, B, ..]
    f32 = 64 * 2.0 ** -24
    names = ["o", "final", "dq", "dk", "dv", "dg", "dbeta", "dstate"]
    for i, u in enumerate(wide):
        w = torch.cat([h[i] for h in halves], which(i)).double()
        bound = 4 * f32 + (0 if u.dtype == torch.float32 else 2 * torch.finfo(dtype).eps / 2)
        assert torch.isfinite(u).all() and float((u.double() - w).norm() / w.norm()) <= bound, ("narrow", names[i])
    some = [0, 2, 16]
    part = [t[some] if i == 5 else t[:, some] for i, t in enumerate(args)]
    ref = heads_reference(part, [lengths[b] for b in some], True, *((go[:, some], gs[some]) if train else ()))
    for i, w in enumerate(ref):
        u = wide[i][some] if which(i) == 0 else wide[i][:, some]
        if u.dtype == torch.float32:
            assert float((u.double() - w).norm() / w.norm()) <= (f32 if i < 2 else 4 * f32), (names[i], float((u.double() - w).norm() / w.norm()))
        else:
            rounded_once(u, w, names[i])


# ------------------------------------------------------------------------------------------ what a caller may do with a result
def test_delta_output_may_be_changed_in_place(cuda):
    """The backward does not need o: a mask multiplied into it in place is differentiated like one multiplied out of place."""
    from speech_amd import ops
    args, go, gs = delta_inputs(70, 2, 2, 2, 16, 24, torch.float32, 12)
    mask = (torch.rand(70, 2, 4, 24, generator=torch.Generator().manual_seed(0)) > 0.3).float().to(cuda)
    grads = []
    for inplace in (True, False):
        xs = [t.to(cuda).requires_grad_(True) for t in args]
        o, f = ops.gated_delta_rule(*xs[:5], state=xs[5], normalize=True)
        o = o.mul_(mask) if inplace else o * mask
        f = f.mul_(0.5) if inplace else f * 0.5
        grads.append(torch.autograd.grad([o, f], xs, [go.to(cuda), gs.to(cuda)]))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("train", [False, True])
def test_delta_without_frames_copies_the_state(cuda, train):
    """The C ABI with T = 0, with and without a place for what a backward would need."""
    from speech_amd import _lib, ops
    h = _lib.lib()
    state, out, some = torch.randn(2, 4, 16, 24, device=cuda), torch.full((2, 4, 16, 24), 7.0, device=cuda), torch.zeros(64, device=cuda)
    strides = ops._host_i64([0] * 15)
    for s0, want in ((state, state), (None, torch.zeros_like(state))):
        saved = some.data_ptr() if train else None
        rc = h.sp_gdr_fwd(None, None, None, None, None, None if s0 is None else s0.data_ptr(), None, strides, 0, 2, 2, 4, 16, 24, 1.0, 0, _lib.SP_F32, None,
                          out.data_ptr(), saved, 256 if train else 0, None, 0, ops.raw_stream(state))
        assert rc == 0, h.sp_last_error()
        assert torch.equal(out, want) and not some.any()


# ------------------------------------------------------------------------------------------ padding has no influence
def _variant(cuda, dtype):
    from speech_amd import net
    torch.manual_seed(3)
    m = net.SRModel(2, 64, 28, 80, 0.0, compute_dtype=dtype, norm="group", rnn="delta").to(cuda)
    with torch.no_grad():
        for blk in m.resnet_layers:
            blk.bn2.weight.uniform_(0.5, 1.0)
            blk.bn1.bias.uniform_(-0.3, 0.3)
            blk.bn2.bias.uniform_(-0.3, 0.3)
    return m


def test_an_utterance_does_not_see_its_batch(cuda):
    """Group norm and delta layers, f32 evaluation: an utterance's logits in a padded batch are those that it has by itself.  Both are within
    f32 rounding of the exact ones: 4096 half steps for the conv stack and 2048 for each layer (test_gpu_operators), twice."""
    from speech_amd import net
    m = _variant(cuda, torch.float32).eval()
    lengths = [90, 61, 40, 3, 0, 90, 1]
    spec = torch.rand(len(lengths), 1, 80, 90, device=cuda)
    L = torch.tensor(lengths, device=cuda)
    with torch.no_grad():
        batch = m(spec, L)
        for b, n in enumerate(lengths):
            if n:
                alone = m(spec[b:b + 1, :, :, :n], L[b:b + 1])
                k = net.out_frames(n)
                assert alone.shape[1] == k
                assert float((batch[b, :k] - alone[0]).norm() / alone.norm()) <= 2 * (4096 + 2 * 2048) * 2.0 ** -24, n
        assert torch.isfinite(batch).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=ids)
def test_padding_holds_anything(cuda, dtype):
    """What lies behind the utterances' frames reaches neither loss nor gradients, not even as NaN.  (The layer norms' and the convolutions'
    parameter gradients are summed with float atomics: 1024 half steps of their largest value.)"""
    m = _variant(cuda, dtype).train()
    lengths = torch.tensor([90, 61, 40, 25], dtype=torch.int32, device=cuda)
    labels = torch.randint(1, 29, (4, 6), generator=torch.Generator().manual_seed(0)).to(cuda)
    ll = torch.tensor([6, 4, 5, 2], dtype=torch.int32, device=cuda)
    spec = torch.rand(4, 1, 80, 90, device=cuda)
    out = []
    for fill in (0.0, 3.0, float("nan"), float("inf")):
        x = spec.clone()
        for b, n in enumerate(lengths.tolist()):
            x[b, :, :, n:] = fill
        m.zero_grad()
        loss = m.ctc_loss(x, labels, ll, lengths=lengths)
        loss.backward()
        out.append((loss.detach(), {n: p.grad.clone() for n, p in m.named_parameters()}))
    for loss, grads in out[1:]:
        assert torch.equal(loss, out[0][0]) and torch.isfinite(loss)
        for n, g in grads.items():
            w = out[0][1][n]
            assert torch.isfinite(g).all() and float((g - w).abs().max()) <= 1024 * 2.0 ** -24 * float(w.abs().max()), n


def test_ctc_scores_own_frames(cuda):
    """The loss of utterances with lengths is CTC over their own encoder frames, in 64 bits from the model's logits."""
    from speech_amd import net
    m = _variant(cuda, torch.float32).eval()
    lengths = torch.tensor([90, 61, 40, 4], device=cuda)
    labels = torch.randint(1, 29, (4, 6), generator=torch.Generator().manual_seed(1)).to(cuda)
    ll = torch.tensor([6, 4, 5, 4], device=cuda)                  # the last one needs more frames than its two: scored over the batch's
    spec = torch.rand(4, 1, 80, 90, device=cuda)
    with torch.no_grad():
        logits = m(spec, lengths).double().cpu()
        loss = m.ctc_loss(spec, labels, ll.int(), lengths=lengths)
        assert torch.equal(loss, m.ctc_loss(spec, labels.cpu(), ll.int().cpu(), lengths=lengths))      # labels from wherever they are
    own = net.score_frames(lengths, labels, ll, logits.shape[1]).cpu()
    assert own.tolist() == [45, 31, 20, 45]
    want = torch.nn.functional.ctc_loss(logits.log_softmax(-1).transpose(0, 1), labels.cpu(), own.long(), ll.cpu(), 0, "mean")
    assert float(loss) == pytest.approx(float(want), rel=1e-5)


def test_commands_hand_the_lengths_on(cuda, monkeypatch):
    """Loaders of the variants carry the clips' frames, training and evaluation give them to the model; the default model's carry none."""
    from speech_amd import data, net, ops, train
    from speech_amd.scripts import eval_dataset as ev
    clips = data.SyntheticSorted(8, 4, seed=3, max_s=2.0)
    hp = dict(batch_size=4, synthetic=True, synthetic_clips=8, steps=1, num_workers=0, multiplier=1)
    for variant in (dict(norm="group", rnn="delta"), dict(norm="batch", rnn="sru")):
        loader, _, evals = train.build_loaders(dict(hp, **variant), 0, 1)
        for x in (loader, evals[0][1]):
            batch = next(iter(x))
            assert len(batch) == (4 if variant["norm"] == "group" else 3)
            if len(batch) == 4:
                assert batch[3].dtype == torch.int32 and int(batch[3].max()) == batch[0].shape[-1]
    assert data.collate_fn(clips[0], "valid", frames=True)[3].tolist() == [ops.num_frames(n) for n in clips.samples[:4]]
    m, seen = _variant(cuda, torch.float32), []
    encode = net.SRModel.encode
    monkeypatch.setattr(net.SRModel, "encode", lambda self, x, lengths=None: (seen.append(None if lengths is None else lengths.tolist()), encode(self, x, lengths))[1])
    frames = [ops.num_frames(n) for n in clips.samples]
    opt = train.FlatAdam(m.parameters(), lr=1e-3)
    from types import SimpleNamespace
    pairs = train.FeaturizingLoader(torch.utils.data.DataLoader(clips, batch_size=None, collate_fn=lambda b: b), "valid", True)
    train.train(4, m, pairs, opt, SimpleNamespace(step=lambda: None), 0, SimpleNamespace(step=lambda: None), 2.0, max_steps=1, log=lambda *a: None)
    assert seen == [frames[:4]]
    train.eval_dataset(m, pairs, "valid", log=lambda *a: None)
    ev.test("synthetic", 4, m, ev.build_loader(clips, None, 0, True), log=lambda *a: None)
    assert seen[1:] == [frames[:4], frames[4:]] * 2


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32, torch.uint8], ids=ids)
def test_lengths_of_any_type_are_clamped(cuda, dtype):
    """Values beyond the tensor mean all of its frames, also those that 32 bits do not hold."""
    from speech_amd import ops
    x, w = torch.randn(3, 2, 7, 16, device=cuda), torch.ones(16, device=cuda)
    args, _, _ = delta_inputs(7, 3, 2, 1, 16, 16, torch.float32, 1, state=False)
    qkv = [t.to(cuda) for t in args[:5]]
    big = {torch.int64: (1 << 32) + 2, torch.int32: (1 << 31) - 1, torch.uint8: 255}[dtype]
    low = {torch.int64: -(1 << 32) + 2, torch.int32: -(1 << 31), torch.uint8: 0}[dtype]
    a, b = torch.tensor([big, 3, low], dtype=dtype, device=cuda), torch.tensor([7, 3, 0], device=cuda)
    assert torch.equal(ops.group_norm(x, w, w, 4, lengths=a), ops.group_norm(x, w, w, 4, lengths=b))
    for u, v in zip(ops.gated_delta_rule(*qkv, lengths=a), ops.gated_delta_rule(*qkv, lengths=b)):
        assert torch.equal(u, v)


def test_layer_step_refuses_before_it_touches_the_state(cuda):
    """A training-mode layer with dropout has no single-frame form."""
    from speech_amd import net
    layer = net.GatedDeltaLayer(64, 64, heads=4, dk=16, dropout=0.1, bidirectional=False).to(cuda).train()
    state = torch.zeros(2, 4, 16, 16, device=cuda)
    with pytest.raises(RuntimeError, match="evaluation"):
        layer.step(torch.randn(2, 64, device=cuda), state)
    assert not state.any()
    layer.eval().step(torch.randn(2, 64, device=cuda), state)
    assert state.any()


@pytest.mark.parametrize("dtype", DTYPES, ids=ids)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("T,at,train", [(12, 5, False), (150, 70, False), (150, 70, True)])
def test_delta_non_finite_values_stay_in_their_head(cuda, dtype, bad, T, at, train):
    """An infinity or NaN in one frame of one head: other heads and utterances, forwards and backwards, and the chunks in front of its own (few
    frames: all frames in front of it) are what they are without it, bit for bit; one in a column of v stays in that column of o."""
    from speech_amd import ops
    args, go, gs = delta_inputs(T, 3, 4, 1, 16, 24, dtype, 31)
    lengths = torch.tensor([T, T - 1, T], device=cuda)

    def run(which, index):
        xs = [t.clone() for t in args]
        if which is not None:
            xs[which][index] = bad
        xs = [t.to(cuda).requires_grad_(train) for t in xs]
        o, f = ops.gated_delta_rule(*xs[:5], state=xs[5], lengths=lengths, normalize=True, bidirectional=True)
        g = torch.autograd.grad([o, f], xs, [go.to(cuda), gs.to(cuda)]) if train else ()
        return o.detach(), f.detach(), g
    o, f, g = run(None, None)
    others = [b * 4 + h for b in range(3) for h in range(4) if (b, h) not in ((1, 0), (1, 2))]
    flat = lambda t: t.flatten(1, 2)[:, others]      # noqa: E731
    front = at if T <= 12 else 64                      # frames of a forward head that do not meet it
    behind = at + 1 if T <= 12 else T - 1 - 64         # of a head that walks backwards, from the utterance's end
    for which, index in ((0, (at, 1, [0, 2])), (1, (at, 1, [0, 2])), (3, (at, 1, [0, 2])), (4, (at, 1, [0, 2]))):
        if which == 3 and bad > 0:
            continue                                    # a gate of +inf is no decay
        p, e, d = run(which, index)
        assert torch.equal(flat(p), flat(o)) and torch.equal(e.flatten(0, 1)[others], f.flatten(0, 1)[others])
        assert torch.equal(p[:front, 1, 0], o[:front, 1, 0]) and torch.equal(p[behind:, 1, 2], o[behind:, 1, 2])
        for x, y in zip(d[:5], g[:5]):
            assert torch.equal(flat(x), flat(y))
    p, e, _ = run(2, (at, 1, 0, 7))
    cols = [c for c in range(24) if c != 7]
    assert torch.equal(p[..., cols], o[..., cols]) and torch.equal(e[..., cols], f[..., cols])


@pytest.mark.parametrize("norm,rnn", [("group", "sru"), ("batch", "delta")])
def test_mixed_variants_take_lengths(cuda, norm, rnn):
    """Group norm in front of SRU layers clears the padding; delta layers behind BatchNorm walk own frames.  A training pass and an evaluation."""
    from speech_amd import convstack, net, ops
    torch.manual_seed(7)
    m = net.SRModel(2, 64, 28, 80, 0.0, compute_dtype=torch.bfloat16, norm=norm, rnn=rnn).to(cuda)
    lengths = torch.tensor([60, 31, 0], device=cuda)
    labels, ll = torch.randint(1, 29, (3, 4), device=cuda), torch.tensor([4, 3, 0], dtype=torch.int32, device=cuda)
    x = torch.rand(3, 1, 80, 60, device=cuda)
    m.train()
    loss = m.ctc_loss(x, labels, ll, lengths=lengths)
    loss.backward()
    assert torch.isfinite(loss) and all(torch.isfinite(p.grad).all() for p in m.parameters() if p.grad is not None)
    m.eval()
    with torch.no_grad():
        got = m.encode(x, lengths)
        if norm == "group":
            dirty = x.clone()
            dirty[1, :, :, 31:], dirty[2] = float("nan"), float("inf")
            assert torch.equal(m.encode(dirty, lengths), got)
        else:
            h = convstack.conv_stack(x, m.cnn, list(m.resnet_layers), False).to(torch.bfloat16)
            h, _ = m.delta_layers(h, torch.tensor([30, 16, 0], device=cuda))
            assert torch.equal(ops.layer_norm(h, m.classifier[0].weight, m.classifier[0].bias, m.classifier[0].eps), got)
