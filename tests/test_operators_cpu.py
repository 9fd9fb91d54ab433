"""Refusals of the encoder operators (group normalisation, counter-based dropout, gated delta rule) and the parts that need no GPU: every
check of the C ABI happens on the host before anything is launched, so the addresses here are never followed."""
import ctypes

import numpy as np
import pytest
import torch

P = 4096          # an aligned address that is never read


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.fixture(scope="module")
def h():
    from speech_amd import _lib
    return _lib.lib()


def _gn(h, N=2, F=3, T=4, C=32, G=8, act=0, dtype=0, x=P, gamma=P, mean=None, rstd=None, strides="ok", ws=P, nws=1 << 20):
    st = i64(*([F * T * C, T * C, C] * 3)) if strides == "ok" else strides
    return h.sp_groupnorm_fwd(x, None, gamma, P, None, st, N, F, T, C, G, 1e-5, act, dtype, P, mean, rstd, ws, nws, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(C=30), -1, b"multiple of G"), (dict(G=0), -1, b"multiple of G"), (dict(C=4096, G=1), -1, b"at most"), (dict(act=3), -1, b"act"),
    (dict(dtype=7), -1, b"dtype"), (dict(N=-1), -1, b"shape"), (dict(N=1 << 23), -1, b"shape"), (dict(x=None), -1, b"null"),
    (dict(gamma=None), -1, b"null"), (dict(mean=P), -1, b"together"), (dict(strides=None), -1, b"strides"), (dict(nws=8), -2, b"workspace"),
    (dict(ws=None), -2, b"workspace"),
])
def test_groupnorm_refuses(h, kw, code, text):
    assert _gn(h, **kw) == code and text in h.sp_last_error()


def test_groupnorm_empty_and_workspace(h):
    assert _gn(h, N=0) == 0 and _gn(h, T=0) == 0
    assert h.sp_groupnorm_workspace_bytes(24032, 1, 1, 1024, 8, 0) == 0          # one position a sample: nothing is kept between kernels
    assert h.sp_groupnorm_workspace_bytes(32, 40, 751, 32, 8, 1) > h.sp_groupnorm_workspace_bytes(32, 40, 751, 32, 8, 0) > 0
    assert h.sp_groupnorm_workspace_bytes(2, 1, 4, 30, 8, 0) == 0                # a shape that every call refuses


@pytest.mark.parametrize("kw,text", [
    (dict(p=-0.1), b"outside"), (dict(p=1.5), b"outside"), (dict(p=float("nan")), b"outside"), (dict(rows=-1), b"shape"), (dict(period=1 << 35), b"shape"),
    (dict(dtype=9), b"dtype"), (dict(rng=None), b"rng"), (dict(x=None), b"null"),
])
def test_dropout_refuses(h, kw, text):
    a = dict(x=P, rows=1, period=64, p=0.1, rng=P, dtype=0)
    a.update(kw)
    assert h.sp_dropout(a["x"], None, a["rows"], a["period"], a["p"], a["rng"], 0, a["dtype"], P, None, None) == -1 and text in h.sp_last_error()


def _gdr(h, T=40, B=2, Hk=2, H=4, dk=64, dv=64, flags=0, dtype=2, q=P, strides=None, state=None, saved=None, nsaved=0, ws=P, nws=1 << 40, scale=1.0):
    st = strides or i64(*([B * Hk * dk, Hk * dk, dk] * 2 + [B * H * dv, H * dv, dv] + [B * H, H, 1] * 2))
    return h.sp_gdr_fwd(q, P, P, P, P, state, None, st, T, B, Hk, H, dk, dv, scale, flags, dtype, P, P, saved, nsaved, ws, nws, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(H=3), -1, b"multiple of Hk"), (dict(Hk=0), -1, b"bad shape"), (dict(dk=60), -1, b"multiples of 8"), (dict(dk=136), -1, b"multiples of 8"),
    (dict(dv=4), -1, b"multiples of 8"), (dict(T=-1), -1, b"bad shape"), (dict(flags=8), -1, b"flags"), (dict(Hk=1, flags=2), -1, b"even"),
    (dict(dtype=5), -1, b"dtype"), (dict(q=None), -1, b"null"), (dict(q=P + 8), -1, b"aligned"), (dict(state=P + 4), -1, b"aligned"),
    (dict(nws=64), -2, b"workspace"), (dict(ws=None), -2, b"workspace"), (dict(saved=P, nsaved=64), -2, b"saved"), (dict(B=1 << 20), -1, b"exceed"),
    (dict(strides=i64(*([1 << 24, 128, 64] * 2 + [512, 256, 64] + [8, 4, 1] * 2))), -1, b"from frame to frame"),
    (dict(strides=i64(*([260, 128, 64] * 2 + [512, 256, 64] + [8, 4, 1] * 2))), -1, b"aligned"),
])
def test_gated_delta_refuses(h, kw, code, text):
    assert _gdr(h, **kw) == code and text in h.sp_last_error()


def test_gated_delta_backward_refuses(h):
    st = i64(*([256, 128, 64] * 2 + [512, 256, 64] + [8, 4, 1] * 2 + [512, 256, 64]))

    def call(T=40, scale=1.0, go=P, saved=P, nsaved=1 << 40, nws=1 << 40):
        return h.sp_gdr_bwd(P, P, P, P, P, None, st, T, 2, 2, 4, 64, 64, scale, 0, 2, P, saved, nsaved, go, None, P, P, P, P, P, None, P, nws, None)
    assert call(scale=0.0) == -1 and b"scale" in h.sp_last_error()
    assert call(T=0) == -1 and b"T=0" in h.sp_last_error()
    assert call(go=None) == -1 and b"null" in h.sp_last_error()
    assert call(nsaved=16) == -2 and call(nws=16) == -2


def test_no_cpu_path():
    from speech_amd import _lib, ops
    x, w = torch.zeros(2, 8), torch.ones(8)
    rng = torch.zeros(2, dtype=torch.int64)
    q, g, s = torch.zeros(3, 2, 2, 8), torch.zeros(3, 2, 2), torch.zeros(2, 2, 8, 8)
    for call in (lambda: ops.group_norm(x, w, w, 2), lambda: ops.dropout(x, 0.1, rng), lambda: ops.gated_delta_rule(q, q, q, g, g),
                 lambda: ops.gated_delta_step(q[0], q[0], q[0], g[0], g[0], s)):
        with pytest.raises(_lib.SpeechHipError, match="CUDA"):
            call()


def philox(counter, key):
    """Philox4x32-10 on Python integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def test_philox_known_answers():
    """The published known answers of the generator (all zeros, all ones), so that the statement the GPU tests use is the generator."""
    f = 0xFFFFFFFF
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_model_variants_check_their_arguments():
    from speech_amd import net
    with pytest.raises(ValueError, match="norm"):
        net.SRModel(2, 64, 28, 80, 0.1, norm="layer")
    with pytest.raises(ValueError, match="rnn"):
        net.SRModel(2, 64, 28, 80, 0.1, rnn="gru")
    with pytest.raises(ValueError, match="projection_size"):
        net.SRModel(2, 64, 28, 80, 0.1, 32, rnn="delta")
    with pytest.raises(ValueError, match="heads"):
        net.GatedDeltaLayer(64, 100)
    with pytest.raises(ValueError, match="both directions"):
        net.GatedDeltaLayer(64, 24, heads=3)
    keys = net.SRModel(2, 64, 28, 80, 0.1, norm="group", rnn="delta").state_dict()
    assert "delta_layers.dropout_state" in keys and "resnet_layers.0.bn1.weight" in keys and "resnet_layers.0.conv1.bias" not in keys
    # the model of the reference keeps its layout
    assert not any(k.startswith("delta") for k in net.SRModel(2, 64, 28, 80, 0.1).state_dict())


def test_delta_layers_refuse_wide_heads_and_reseed():
    from speech_amd import net
    with pytest.raises(ValueError, match="at most 128 wide"):
        net.GatedDeltaLayer(64, 2048, heads=8)
    with pytest.raises(ValueError, match="at most 128 wide"):
        net.GatedDeltaLayer(64, 1024, heads=8, dk=136)
    assert net.SRModel(1, 1024, 28, 80, 0.0, rnn="delta").delta_layers.layers[0].heads == 16
    m = net.GatedDelta(64, 64, 1, 0.1)
    m.dropout_state[1] = 7
    m.load_state_dict(net.GatedDelta(64, 64, 1, 0.1).state_dict())          # another rank's seed and step
    m.reseed(12345)
    assert m.dropout_state.tolist() == [12345, 0]


def test_train_flags():
    from speech_amd import train
    hp = train.parse_args(["--synthetic", "--norm", "group", "--rnn", "delta"])
    assert hp["norm"] == "group" and hp["rnn"] == "delta"
    assert train.parse_args([])["norm"] == "batch" and train.parse_args([])["rnn"] == "sru"


def test_group_block_is_the_plain_group_norm():
    """ResidualBlock's plain statement with groups: torch's GroupNorm in the place of BatchNorm, no convolution bias."""
    from speech_amd import net
    torch.manual_seed(0)
    b = net.ResidualBlock(32, 32, 5, groups=8)
    with torch.no_grad():
        b.bn2.weight.fill_(0.5)
    x = torch.randn(2, 32, 6, 7)
    y = torch.relu(torch.nn.functional.group_norm(b.conv1(x), 8, b.bn1.weight, b.bn1.bias))
    y = torch.relu(torch.nn.functional.group_norm(b.conv2(y), 8, b.bn2.weight, b.bn2.bias) + x)
    np.testing.assert_allclose(b(x).detach().numpy(), y.detach().numpy(), rtol=1e-5, atol=1e-5)
