"""Edges of the encoder operators that need no GPU: what the C ABI checks on the host before anything is launched (no address is followed),
the build's dependencies, the models' arguments."""
import ctypes
import os
import time

import pytest

P = 4096          # an aligned address that is never read


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.fixture(scope="module")
def h():
    from speech_amd import _lib
    return _lib.lib()


STRIDES = i64(*([256, 128, 64] * 2 + [512, 256, 64] + [8, 4, 1] * 2 + [512, 256, 64]))


def _gdr_bwd(h, o=P, saved=P, go=P, gq=P, gk=P, gv=P, ws=P, nws=1 << 40):
    return h.sp_gdr_bwd(P, P, P, P, P, None, STRIDES, 40, 2, 2, 4, 64, 64, 1.0, 0, 2, o, saved, 1 << 40, go, None, gq, gk, gv, P, P, None, ws, nws, None)


def test_gated_delta_backward_does_not_ask_for_o(h):
    assert _gdr_bwd(h, o=None, nws=16) == -2 and b"workspace" in h.sp_last_error()      # past the check of addresses, refused for its workspace


@pytest.mark.parametrize("name", ["saved", "gq", "gk", "gv", "ws"])
def test_gated_delta_backward_asks_for_aligned_buffers(h, name):
    """They are read and written 16 bytes at a time."""
    assert _gdr_bwd(h, **{name: P + 8}) == -1 and b"aligned" in h.sp_last_error()


@pytest.mark.parametrize("name", ["saved", "ws", "state_out", "o"])
def test_gated_delta_forward_asks_for_aligned_buffers(h, name):
    a = dict(saved=P if name == "saved" else None, ws=P, state_out=P, o=P)
    a[name] = P + 4
    assert h.sp_gdr_fwd(P, P, P, P, P, None, None, STRIDES, 40, 2, 2, 4, 64, 64, 1.0, 0, 2, a["o"], a["state_out"], a["saved"], 1 << 40, a["ws"], 1 << 40,
                        None) == -1 and b"aligned" in h.sp_last_error()


def test_gated_delta_grid_is_limited_as_documented(h):
    assert h.sp_gdr_workspace_bytes(64 * 59, 8192, 8, 8, 8, 8, 2, 0) > 0        # 65536 * (59 + 4) = 2^22 - 2^16
    assert h.sp_gdr_workspace_bytes(64 * 60, 8192, 8, 8, 8, 8, 2, 0) == 0 and b"grid" in h.sp_last_error()


def test_build_follows_its_flags(tmp_path, monkeypatch):
    """An object is built again when its source, a header or the file that holds the compiler's flags is newer."""
    from speech_amd import build
    src, obj = tmp_path / "csrc", tmp_path / "build"
    src.mkdir()
    files = {n: src / n for n in ("a.hip", "b.hip", "common.h")}
    flags, lib = tmp_path / "build.py", tmp_path / "lib.so"
    for p in (*files.values(), flags):
        p.write_text("x")
    compiled = []

    def compile_(name):
        compiled.append(name)
        (obj / (name[:-4] + ".o")).write_text("o")

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def link(cmd, **kw):
        lib.write_text("lib")
        return Done
    for name, value in (("CSRC", str(src)), ("OBJDIR", str(obj)), ("LIB", str(lib)), ("SELF", str(flags)), ("_compile", compile_)):
        monkeypatch.setattr(build, name, value)
    monkeypatch.setattr(build.subprocess, "run", link)

    def newer(p):
        t = time.time() + 100 * (len(compiled) + 1)
        os.utime(p, (t, t))

    def again():
        n = len(compiled)
        build.build(verbose=False)
        return sorted(compiled[n:])
    assert again() == ["a.hip", "b.hip"]
    assert again() == []
    newer(files["a.hip"])
    assert again() == ["a.hip"]
    for p in (src / "a.hip", obj / "a.o"):
        os.utime(p, (time.time(), time.time()))
    assert again() == []
    newer(flags)
    assert again() == ["a.hip", "b.hip"]


def test_the_default_model_takes_no_lengths():
    import torch
    from speech_amd import net
    x = torch.zeros(2, 1, 80, 20)
    m = net.SRModel(1, 64, 28, 80, 0.0)
    assert not m.takes_lengths
    for call in (m.encode, m):
        with pytest.raises(ValueError, match="padding"):
            call(x, torch.tensor([20, 10]))
    for kw in (dict(norm="group"), dict(rnn="delta")):
        m = net.SRModel(1, 64, 28, 80, 0.0, **kw)
        assert m.takes_lengths
        for bad in (torch.tensor([20]), torch.tensor([20.0, 10.0]), torch.tensor([True, False])):
            with pytest.raises(ValueError, match="whole numbers"):
                m(x, bad)


def test_frames_that_ctc_scores():
    """Own frames, or the batch's where a transcript needs more: its labels and a blank between equal neighbours."""
    import torch
    from speech_amd import net
    labels = torch.tensor([[1, 1, 2, 2], [1, 2, 3, 9], [4, 4, 4, 0], [5, 0, 0, 0]])
    n = torch.tensor([4, 3, 3, 1], dtype=torch.int32)                # needs 6, 3, 5, 1
    assert net.score_frames(torch.tensor([11, 5, 8, 1]), labels, n, 30).tolist() == [6, 3, 30, 1]
    assert net.score_frames(torch.tensor([10, 4, 9, 0], dtype=torch.int32), labels, n, 30).tolist() == [30, 30, 5, 30]
    assert net.score_frames(torch.tensor([99, 99], dtype=torch.uint8), labels[:2, :0], n[:2] * 0, 30).tolist() == [30, 30]
