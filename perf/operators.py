"""Cases of the encoder operators: group normalisation with an activation, counter-based dropout and the gated delta rule.

``run`` computes a case in plain torch arithmetic, or, with ``own`` set, through ``speech_amd.ops``; ``exact`` restates each operator in
64 bits.  Sizes are those of the acoustic encoder (32 utterances of 15 s: 751 frames of 32 channels x 40 bands, 1024 features, 8 heads)
and generic ones around them.
"""
import math

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # ---- group normalisation, channels last [N, F, T, C] ----
        # a residual block of the conv stack in training, 32 x 15 s
        dict(name="gn_train_block", op="gn", dtype="bf16", N=32, F=40, T=751, C=32, G=8, act="silu", res=True, ragged=False, train=True),
        # the output norm of a recurrent encoder layer: one group per head, every frame a sample of its own
        dict(name="gn_train_heads", op="gn", dtype="bf16", N=24032, F=1, T=1, C=1024, G=8, act="silu", res=False, ragged=False, train=True),
        # evaluation of a ragged batch in the half-precision inference type
        dict(name="gn_infer_ragged", op="gn", dtype="f16", N=13, F=40, T=333, C=32, G=4, act="relu", res=True, ragged=True, train=False),
        # one second of one utterance, full precision: latency
        dict(name="gn_infer_short", op="gn", dtype="f32", N=1, F=40, T=50, C=32, G=8, act="relu", res=False, ragged=False, train=False),
        # ---- dropout ----
        # residual dropout of an encoder layer in training
        dict(name="drop_train", op="drop", dtype="bf16", T=751, B=32, C=1024, p=0.1, res=True, shared=False, train=True),
        # variational dropout (one mask for all frames) at an odd width
        dict(name="drop_shared", op="drop", dtype="f32", T=333, B=7, C=485, p=0.35, res=False, shared=True, train=True),
        # ---- gated delta rule [T, B, H, d] ----
        # an encoder layer in training, 32 x 15 s, both directions
        dict(name="delta_train", op="delta", dtype="bf16", T=751, B=32, Hk=8, r=1, dk=64, dv=128, ragged=False, norm=True, bidir=True, state=False, train=True),
        # training in full precision: shared key heads, odd widths, ragged, with a state handed in
        dict(name="delta_train_f32", op="delta", dtype="f32", T=301, B=5, Hk=2, r=3, dk=40, dv=72, ragged=True, norm=False, bidir=False, state=True, train=True),
        # evaluation of 30 s utterances with the widest keys
        dict(name="delta_infer_long", op="delta", dtype="bf16", T=1501, B=16, Hk=8, r=1, dk=128, dv=128, ragged=True, norm=True, bidir=False, state=False, train=False),
        # a streaming recogniser: sixteen new frames of one session
        dict(name="delta_stream_16", op="delta", dtype="bf16", T=16, B=1, Hk=8, r=1, dk=64, dv=128, ragged=False, norm=True, bidir=False, state=True, train=False),
        # one new frame for 64 sessions at once
        dict(name="delta_step_64", op="step", dtype="bf16", B=64, Hk=8, r=1, dk=128, dv=128, norm=True),
        # one new frame of one session: latency
        dict(name="delta_step_1", op="step", dtype="f16", B=1, Hk=4, r=2, dk=64, dv=128, norm=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["gn", "gn", "drop", "delta", "delta", "step"])
    dt = rng.choice(["bf16", "f16", "f32"])
    if kind == "gn":
        if rng.random() < 0.3:      # one sample a frame
            C = 8 * _log(rng, 4, 128)
            G = rng.choice([g for g in (1, 2, 4, 8, 16) if C % g == 0])
            N, F, T = min(_log(rng, 50, 24000), 24_000_000 // C), 1, 1
        else:
            C = rng.choice([8, 20, 32, 48, 64, 96, 160, 256])
            G = rng.choice([g for g in (1, 2, 4, 8, 16, 32) if C % g == 0])
            N, F, T = _log(rng, 1, 32), rng.choice([1, 5, 20, 40]), _log(rng, 1, 1501)
            T = max(1, min(T, 20_000_000 // (N * F * C)))
        train = rng.random() < 0.5
        return dict(op="gn", dtype=dt, N=N, F=F, T=T, C=C, G=G, act=rng.choice(["silu", "none"] if train else ["relu", "silu", "none"]),
                    res=rng.random() < 0.5, ragged=F * T > 1 and rng.random() < 0.4, train=train)
    if kind == "drop":
        C, B = _log(rng, 3, 1300), _log(rng, 1, 40)
        T = max(1, min(_log(rng, 1, 1501), 20_000_000 // (B * C)))
        return dict(op="drop", dtype=dt, T=T, B=B, C=C, p=round(rng.uniform(0.02, 0.6), 3), res=rng.random() < 0.5, shared=rng.random() < 0.4, train=rng.random() < 0.7)
    r = rng.choice([1, 1, 2, 3])
    dk, dv = 8 * rng.randint(1, 16), 8 * rng.randint(1, 16)
    if kind == "step":
        return dict(op="step", dtype=dt, B=_log(rng, 1, 64), Hk=rng.choice([1, 2, 4]), r=r, dk=dk, dv=dv, norm=rng.random() < 0.6)
    train = rng.random() < 0.5
    T, Hk = _log(rng, 1, 1501), rng.choice([1, 2, 4])
    B = max(1, min(_log(rng, 1, 32), 60_000 // (T * Hk * r)))
    return dict(op="delta", dtype=dt, T=T, B=B, Hk=Hk, r=r, dk=dk, dv=dv, ragged=rng.random() < 0.5, norm=rng.random() < 0.6,
                bidir=Hk > 1 and rng.random() < 0.4, state=rng.random() < 0.5, train=train)


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] == "gn":
        n = case["N"] * case["F"] * case["T"] * case["C"]
        passes = 2 + case["res"] + ((2 + case["res"]) if case["train"] else 0)
        return {"bytes": n * e * passes + 16 * case["C"], "flops": n * (30 if case["train"] else 12)}
    if case["op"] == "drop":
        n = case["T"] * case["B"] * case["C"]
        return {"bytes": n * e * (2 + case["res"] + (2 if case["train"] else 0)), "flops": n * (30 if case["train"] else 15)}
    T = case.get("T", 1)
    H, dk, dv = case["Hk"] * case["r"], case["dk"], case["dv"]
    rows = T * case["B"]
    qkv = rows * e * (2 * case["Hk"] * dk + H * dv) + rows * H * 8
    state = case["B"] * H * dk * dv * 4
    if case["op"] == "step":
        return {"bytes": qkv + rows * H * dv * e + 2 * state, "flops": 6 * rows * H * dk * dv}
    b = qkv + rows * H * dv * e + state * (1 + case["state"])
    f = 6 * rows * H * dk * dv
    if case["train"]:           # dO read, the gradients written, the state's gradients read and written
        b += rows * H * dv * e + qkv + state * (1 + case["state"])
        f *= 3
    return {"bytes": b, "flops": f}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _lengths(g, n, T, dev, ragged):
    if not ragged:
        return None
    v = torch.randint(1, T + 1, (n,), generator=g, device=dev)
    v[torch.randint(0, n, (1,), generator=g, device=dev)] = T
    if n > 3:
        v[torch.randint(0, n, (1,), generator=g, device=dev)] = 0       # an utterance of which nothing is left
    return v.to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) % (1 << 62))
    dt = _DT[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * std).to(dt)

    s = {"case": dict(case)}
    if case["op"] == "gn":
        N, F, T, C = (case[k] for k in "NFTC")
        s["x"] = (torch.randn(N, F, T, C, generator=g, device=dev) * 1.5 + torch.randn(C, generator=g, device=dev)).to(dt)
        s["w"] = 1 + 0.2 * torch.randn(C, generator=g, device=dev)
        s["b"] = 0.2 * torch.randn(C, generator=g, device=dev)
        s["res"] = normal(N, F, T, C) if case["res"] else None
        s["gy"] = normal(N, F, T, C) if case["train"] else None
        s["lengths"] = _lengths(g, N, T, dev, case["ragged"])
    elif case["op"] == "drop":
        T, B, C = case["T"], case["B"], case["C"]
        s["x"] = normal(T, B, C)
        s["res"] = normal(T, B, C) if case["res"] else None
        s["gy"] = normal(T, B, C) if case["train"] else None
        s["rng"] = torch.tensor([(int(seed) * 0x9E3779B97F4A7C15 + 12345) % (1 << 62), int(seed) % 1000], dtype=torch.int64, device=dev)
        s["stream"] = 3
    else:
        T, B, Hk, r, dk, dv = case.get("T", 1), case["B"], case["Hk"], case["r"], case["dk"], case["dv"]
        H = Hk * r
        lead = (B,) if case["op"] == "step" else (T, B)
        s["q"], s["k"], s["v"] = normal(*lead, Hk, dk), normal(*lead, Hk, dk), normal(*lead, H, dv)
        if not case["norm"]:        # keys that the producer has brought to unit length
            for n in "qk":
                s[n] = (s[n].float() / s[n].float().square().sum(-1, keepdim=True).sqrt()).to(dt)
        # decays from a thousandth to two nats a frame, as a softplus gate with a rate per head gives them
        rate = torch.exp(torch.empty(H, device=dev).uniform_(math.log(0.005), 0.0, generator=g))
        s["g"] = -rate * torch.nn.functional.softplus(torch.randn(*lead, H, generator=g, device=dev))
        s["beta"] = torch.sigmoid(torch.randn(*lead, H, generator=g, device=dev))
        s["state"] = torch.randn(B, H, dk, dv, generator=g, device=dev) * 0.3 if case["op"] == "step" or case["state"] else None
        if case["op"] == "delta":
            s["lengths"] = _lengths(g, B, T, dev, case["ragged"])
            if case["train"]:
                s["go"] = normal(T, B, H, dv)
                s["gstate"] = torch.randn(B, H, dk, dv, generator=g, device=dev) * 0.1
    if case.get("train"):
        for n in ("x", "w", "b", "res", "q", "k", "v", "g", "beta", "state"):
            if s.get(n) is not None:
                s[n].requires_grad_(True)
    return s


# ----------------------------------------------------------------------------------------------------- the framework's operators
def _run_own(s):
    from speech_amd import ops
    c = s["case"]
    if c["op"] == "gn":
        y = ops.group_norm(s["x"], s["w"], s["b"], c["G"], act=c["act"], residual=s["res"], lengths=s["lengths"])
        if not c["train"]:
            return y
        leaves = [t for t in (s["x"], s["w"], s["b"], s["res"]) if t is not None]
        return [y.detach(), *torch.autograd.grad(y, leaves, s["gy"])]
    if c["op"] == "drop":
        y = ops.dropout(s["x"], c["p"], s["rng"], s["stream"], residual=s["res"], shared=c["shared"])
        if not c["train"]:
            return y
        return [y.detach(), torch.autograd.grad(y, [s["x"]], s["gy"])[0]]
    if c["op"] == "step":
        return [ops.gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], normalize=c["norm"]), s["state"]]
    o, final = ops.gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], state=s["state"], lengths=s["lengths"], normalize=c["norm"],
                                    bidirectional=c["bidir"])
    if not c["train"]:
        return [o, final]
    leaves = [t for t in (s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"]) if t is not None]
    return [o.detach(), final.detach(), *torch.autograd.grad([o, final], leaves, [s["go"], s["gstate"]])]


# ------------------------------------------------------------------------------------------------------------- the plain forms
def _gn_plain(s):
    c = s["case"]
    with torch.no_grad():
        x = s["x"].float()
        N, F, T, C = x.shape
        G = c["G"]
        w, b = s["w"], s["b"]
        m, cnt = None, float(F * T * (C // G))
        if s["lengths"] is not None:
            m = (torch.arange(T, device=x.device) < s["lengths"][:, None]).view(N, 1, T, 1)
            cnt = (s["lengths"].float() * (F * (C // G))).clamp_min(1.0).view(N, 1, 1, 1, 1)

        def group_mean(t):
            t = t if m is None else torch.where(m, t, 0.0)
            return (t.view(N, F, T, G, C // G).sum((1, 2, 4), keepdim=True) / cnt).expand(N, 1, 1, G, C // G).reshape(N, 1, 1, C)

        d = x - group_mean(x)
        rstd = (group_mean(d * d) + 1e-5) ** -0.5
        xhat = d * rstd
        pre = xhat * w + b
        if s["res"] is not None:
            pre = pre + s["res"].float()
        if c["act"] == "relu":
            y, slope = torch.where(pre > 0, pre, 0.0), (pre > 0).float()
        elif c["act"] == "silu":
            sg = 1 / (1 + torch.exp(-pre))
            y, slope = pre * sg, sg * (1 + pre * (1 - sg))
        else:
            y, slope = pre, 1.0
        if m is not None:
            y = torch.where(m, y, 0.0)
        if not c["train"]:
            return y.to(s["x"].dtype)
        gr = s["gy"].float() * slope
        if m is not None:
            gr = torch.where(m, gr, 0.0)
        dw, db = (gr * xhat).sum((0, 1, 2)), gr.sum((0, 1, 2))
        gw = gr * w
        dx = rstd * (gw - group_mean(gw) - xhat * group_mean(gw * xhat))
        if m is not None:
            dx = torch.where(m, dx, 0.0)
        dt = s["x"].dtype
        return [y.to(dt), dx.to(dt), dw, db] + ([gr.to(dt)] if s["res"] is not None else [])


def _philox_plain(index, seed, step, stream):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC'11) on int64 tensors holding 32-bit words -> four words."""
    M = 0xFFFFFFFF

    def mul(a, b):              # high and low word of a 32 x 32 bit product
        lo16 = (b & 0xFFFF) * a
        up = (b >> 16) * a + (lo16 >> 16)
        return up >> 16, ((up & 0xFFFF) << 16) | (lo16 & 0xFFFF)

    c0, c1 = index & M, (index >> 32) & M
    c2, c3 = (step & M).expand_as(c0), torch.full_like(c0, stream & M)
    k0, k1 = seed & M, (seed >> 32) & M
    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & M, (k1 + 0xBB67AE85) & M
    return c0, c1, c2, c3


def _drop_plain(s):
    c = s["case"]
    with torch.no_grad():
        x = s["x"].float()
        n = x[0].numel() if c["shared"] else x.numel()
        at = torch.arange((n + 7) // 8, device=x.device)
        words = torch.stack(_philox_plain(at, s["rng"][0], s["rng"][1], s["stream"]), -1)
        draws = torch.stack([words & 0xFFFF, words >> 16], -1).view(-1)[:n]      # eight 16-bit draws a counter
        thr = int(round(c["p"] * 65536))
        keep = (draws >= thr).view(x.shape[1:] if c["shared"] else x.shape)
        scale = 65536.0 / (65536 - thr)
        y = torch.where(keep, x * scale, 0.0)
        if s["res"] is not None:
            y = y + s["res"].float()
        if not c["train"]:
            return y.to(s["x"].dtype)
        return [y.to(s["x"].dtype), torch.where(keep, s["gy"].float() * scale, 0.0).to(s["x"].dtype)]


def _turn(t, lengths):
    """[B, H, T, ...] with the second half of the heads reversed in time over each utterance's own frames (its own inverse)."""
    B, H, T = t.shape[:3]
    at = torch.arange(T, device=t.device).expand(B, T)
    n = lengths[:, None] if lengths is not None else T
    at = torch.where(at < n, n - 1 - at, at).view(B, 1, T, *[1] * (t.dim() - 3)).expand(B, H - H // 2, *t.shape[2:])
    return torch.cat([t[:, :H // 2], torch.gather(t[:, H // 2:], 2, at)], 1)


def _delta_heads(s, f):
    """q, k, v, g, beta as [B, H, T, ...] in type f: key heads repeated over their group, normalised and scaled, padding cleared."""
    c = s["case"]
    q, k, v, g, b = (s[n].to(f) for n in ("q", "k", "v", "g", "beta"))
    if c["norm"]:
        q, k = (t * (t.square().sum(-1, keepdim=True) + 1e-6) ** -0.5 for t in (q, k))
    q = q * c["dk"] ** -0.5
    q, k = (t.repeat_interleave(c["r"], 2) for t in (q, k))
    q, k, v, g, b = (t.movedim(0, 2) for t in (q, k, v, g, b))
    if s["lengths"] is not None:
        m = torch.arange(c["T"], device=q.device) < s["lengths"][:, None, None]
        q, k, v = (torch.where(m[..., None], t, 0.0) for t in (q, k, v))
        g, b = (torch.where(m, t, 0.0) for t in (g, b))
    if c["bidir"]:
        q, k, v, g, b = (_turn(t, s["lengths"]) for t in (q, k, v, g, b))
    return q, k, v, g, b


def _delta_out(s, o):
    """[B, H, T, dv] back to [T, B, H, dv], frames behind an utterance's end cleared."""
    if s["case"]["bidir"]:
        o = _turn(o, s["lengths"])
    if s["lengths"] is not None:
        o = torch.where((torch.arange(o.shape[2], device=o.device) < s["lengths"][:, None, None])[..., None], o, 0.0)
    return o.movedim(2, 0).to(s["v"].dtype)


def _delta_chunks(s, L=64):
    """The chunked form: everything but the state's walk is one batched product over all chunks."""
    c = s["case"]
    q, k, v, g, b = _delta_heads(s, torch.float32)
    B, H, T = g.shape
    n = (T + L - 1) // L
    pad = n * L - T

    def cut(t):
        t = torch.cat([t, t.new_zeros(B, H, pad, *t.shape[3:])], 2) if pad else t
        return t.reshape(B * H, n, L, *t.shape[3:])

    q, k, v, g, b = (cut(t) for t in (q, k, v, g, b))
    G = g.cumsum(-1)
    low = torch.ones(L, L, dtype=torch.bool, device=g.device).tril()
    D = torch.exp(torch.where(low, G[..., :, None] - G[..., None, :], -1e30))
    kt = k.transpose(-1, -2).contiguous()
    A = torch.where(low.tril(-1), (k @ kt) * D, 0.0) * b[..., :, None]
    inv, P = torch.eye(L, device=g.device) - A, A @ A
    for _ in range(5):                                       # (I + A)^-1 of a nilpotent A by doubling
        inv, P = inv + inv @ P, P @ P
    V0 = inv @ (b[..., None] * v)
    W = inv @ ((b * torch.exp(G))[..., None] * k)
    att = (q @ kt) * D
    qd = q * torch.exp(G)[..., None]
    last = G[..., -1:]
    kd = (k * torch.exp(last - G)[..., None]).transpose(-1, -2).contiguous()
    end = torch.exp(last)[..., None]
    S = s["state"].reshape(B * H, c["dk"], c["dv"]) if s["state"] is not None else q.new_zeros(B * H, c["dk"], c["dv"])
    out = []
    for i in range(n):
        u = V0[:, i] - W[:, i] @ S
        out.append(qd[:, i] @ S + att[:, i] @ u)
        S = end[:, i] * S + kd[:, i] @ u
    o = torch.cat(out, 1)[:, :T].reshape(B, H, T, c["dv"])
    return _delta_out(s, o), S.view(B, H, c["dk"], c["dv"])


def _delta_plain(s):
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return list(_delta_chunks(s))
    o, final = _delta_chunks(s)
    leaves = [t for t in (s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"]) if t is not None]
    return [o.detach(), final.detach(), *torch.autograd.grad([o, final], leaves, [s["go"], s["gstate"]])]


def _step_plain(s):
    c = s["case"]
    with torch.no_grad():
        q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
        if c["norm"]:
            q, k = (t * (t.square().sum(-1, keepdim=True) + 1e-6) ** -0.5 for t in (q, k))
        q, k = ((t.repeat_interleave(c["r"], 1)[..., None]) for t in (q * c["dk"] ** -0.5, k))
        S = s["state"] * torch.exp(s["g"])[..., None, None]
        u = s["beta"][..., None] * (v - (S * k).sum(-2))
        S = S + k * u[..., None, :]
        s["state"].copy_(S)
        return [(S * q).sum(-2).to(s["v"].dtype), s["state"]]


def run(state):
    if own:
        return _run_own(state)
    return {"gn": _gn_plain, "drop": _drop_plain, "delta": _delta_plain, "step": _step_plain}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- in 64 bits
def _gn_exact(s):
    c = s["case"]
    x, w, b = (s[n].detach().double().requires_grad_(True) for n in ("x", "w", "b"))
    res = s["res"].detach().double().requires_grad_(True) if s["res"] is not None else None
    rows = []
    G = c["G"]
    for n in range(c["N"]) if s["lengths"] is not None else [slice(None)]:
        xn = x[n:n + 1, :, :int(s["lengths"][n])] if s["lengths"] is not None else x
        if xn.numel() == 0:
            rows.append(x[n:n + 1] * 0)
            continue
        parts = xn.unflatten(-1, (G, -1)).permute(0, 3, 1, 2, 4).flatten(2)
        var, mean = torch.var_mean(parts, -1, unbiased=False)
        spread = lambda t: t.repeat_interleave(c["C"] // G, 1)[:, None, None, :]      # noqa: E731
        z = (xn - spread(mean)) / (spread(var) + 1e-5).sqrt() * w + b
        if res is not None:
            z = z + (res[n:n + 1, :, :xn.shape[2]] if s["lengths"] is not None else res)
        z = z.clamp_min(0) if c["act"] == "relu" else z * torch.sigmoid(z) if c["act"] == "silu" else z
        if xn.shape[2] < c["T"]:
            z = torch.cat([z, z.new_zeros(1, c["F"], c["T"] - xn.shape[2], c["C"])], 2)
        rows.append(z)
    y = torch.cat(rows)
    if not c["train"]:
        return y.detach()
    return [y.detach(), *torch.autograd.grad(y, [t for t in (x, w, b, res) if t is not None], s["gy"].double())]


def _drop_exact(s):
    c = s["case"]
    x = s["x"].detach().double().cpu().numpy()
    n = x[0].size if c["shared"] else x.size
    seed, step = (int(v) for v in s["rng"].tolist())
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    at = np.arange((n + 7) // 8, dtype=u)
    ctr = [at & low, at >> half, np.full_like(at, step & 0xFFFFFFFF), np.full_like(at, s["stream"])]
    for rnd in range(10):
        k0, k1 = u((seed + rnd * 0x9E3779B9) & 0xFFFFFFFF), u(((seed >> 32) + rnd * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = u(0xD2511F53) * ctr[0], u(0xCD9E8D57) * ctr[2]
        ctr = [(b >> half) ^ ctr[1] ^ k0, b & low, (a >> half) ^ ctr[3] ^ k1, a & low]
    bits = np.stack(ctr, -1).astype("<u4").view("<u2").reshape(-1)[:n]
    thr = int(round(c["p"] * 65536))
    gain = (bits >= thr).reshape(x.shape[1:] if c["shared"] else x.shape) * (65536.0 / (65536 - thr))
    y = x * gain
    if s["res"] is not None:
        y = y + s["res"].detach().double().cpu().numpy()
    return [torch.from_numpy(y), torch.from_numpy(s["gy"].double().cpu().numpy() * gain)] if c["train"] else torch.from_numpy(y)


def _delta_frames(S, q, k, v, a, b):
    """Frame by frame, straight from the definition: [B, H, n, ...] -> outputs and the state behind the last frame."""
    out = []
    for t in range(q.shape[2]):
        S = S * a[:, :, t, None, None]
        u = (v[:, :, t] - (k[:, :, t, :, None] * S).sum(2)) * b[:, :, t, None]
        S = S + k[:, :, t, :, None] * u[:, :, None, :]
        out.append((q[:, :, t, :, None] * S).sum(2))
    return torch.stack(out, 2), S


def _delta_exact(s):
    from torch.utils.checkpoint import checkpoint
    c = s["case"]
    w = dict(s)
    for n in ("q", "k", "v", "g", "beta", "state"):
        if s[n] is not None:
            w[n] = s[n].detach().double().requires_grad_(c["train"])
    q, k, v, g, b = _delta_heads(w, torch.float64)
    a = torch.exp(g)
    S = w["state"] if w["state"] is not None else q.new_zeros(*g.shape[:2], c["dk"], c["dv"])
    outs = []
    for t in range(0, c["T"], 50):
        part = [x[:, :, t:t + 50] for x in (q, k, v, a, b)]
        o, S = checkpoint(_delta_frames, S, *part, use_reentrant=False) if c["train"] else _delta_frames(S, *part)
        outs.append(o)
    o = _delta_out(w, torch.cat(outs, 2))
    if not c["train"]:
        return [o, S]
    leaves = [w[n] for n in ("q", "k", "v", "g", "beta", "state") if w[n] is not None]
    return [o.detach(), S.detach(), *torch.autograd.grad([o, S], leaves, [s["go"].double(), s["gstate"].double()])]


def _step_exact(s):
    c = s["case"]
    q, k, v, g, b, S = (s[n].double() for n in ("q", "k", "v", "g", "beta", "state"))
    if c["norm"]:
        q, k = q / (q.pow(2).sum(-1, True) + 1e-6).sqrt(), k / (k.pow(2).sum(-1, True) + 1e-6).sqrt()
    q, k = q.repeat_interleave(c["r"], 1) / math.sqrt(c["dk"]), k.repeat_interleave(c["r"], 1)
    S = torch.exp(g)[..., None, None] * S
    S = S + torch.einsum("bhk,bhv->bhkv", k, b[..., None] * (v - torch.einsum("bhk,bhkv->bhv", k, S)))
    return [torch.einsum("bhk,bhkv->bhv", q, S), S]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "step":
        with torch.no_grad():
            return _step_exact(s)
    if case["op"] == "gn" and not case["train"] or case["op"] == "delta" and not case["train"]:
        with torch.no_grad():
            return {"gn": _gn_exact, "delta": _delta_exact}[case["op"]](s)
    return {"gn": _gn_exact, "drop": _drop_exact, "delta": _delta_exact}[case["op"]](s)
