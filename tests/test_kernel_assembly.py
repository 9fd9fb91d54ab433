"""The compiler has lost live registers at the end of loops that end lane by lane: at such an exit it put the copy of a register (to an
accumulation register, in a kernel that needs more than 256) in front of the instruction that turns the lanes on again, so that the copy
wrote nothing.  The assembly of the kernels built here is searched for vector instructions in that place."""
import re
import subprocess

_LABEL = re.compile(r"(\.LBB\d+_\d+):")
_ENDS = re.compile(r"s_cbranch|s_branch|s_endpgm|s_barrier|s_and_saveexec|s_and_b64 exec|s_mov_b64 exec")
_LANES_ON = re.compile(r"s_or_b64 exec, exec,|s_or_saveexec|s_andn2_saveexec")


def lost_writes(assembly):
    """[(kernel, label, instructions)]: vector instructions between a place that no lane need reach and the one that turns lanes on again."""
    found = []
    for f in re.finditer(r"^(\S+):\s*; @\1\n(.*?)\.Lfunc_end", assembly, re.S | re.M):
        lines = [x.split(";")[0].strip() for x in f.group(2).splitlines()]
        joins = {x.split()[1] for x in lines if x.startswith("s_cbranch_execz")}
        for i, line in enumerate(lines):
            label = _LABEL.match(line)
            if not (label and label.group(1) in joins) and not line.startswith("s_cbranch_execnz"):
                continue
            vector = []
            for x in lines[i + 1:]:
                if _LANES_ON.match(x):
                    if vector:
                        found.append((f.group(1), line, vector))
                    break
                if _ENDS.match(x):
                    break
                if re.match(r"v_|ds_|global_|buffer_|scratch_|flat_", x) and not re.match(r"v_(read|write)(first)?lane", x):
                    vector.append(x)
    return found


def test_the_search_finds_a_planted_copy():
    kernel = "k:  ; @k\n s_and_saveexec_b64 s[0:1], vcc\n s_cbranch_execz .LBB0_2\n v_mov_b32 v1, v2\n.LBB0_2:\n{} s_or_b64 exec, exec, s[0:1]\n v_mov_b32 v3, v4\n.Lfunc_end0\n"
    loop = "k:  ; @k\n.LBB0_1:\n s_andn2_b64 exec, exec, s[2:3]\n s_cbranch_execnz .LBB0_1\n{} s_or_b64 exec, exec, s[2:3]\n.Lfunc_end0\n"
    for text in (kernel, loop):
        assert not lost_writes(text.format(""))
        assert [x[2] for x in lost_writes(text.format(" v_accvgpr_write_b32 a48, v47\n"))] == [["v_accvgpr_write_b32 a48, v47"]]


def test_no_kernel_of_the_delta_rule_loses_a_copy(tmp_path):
    """delta.hip holds the library's kernels that need more than 256 registers."""
    from speech_amd import build
    out = tmp_path / "delta.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "-S", "--cuda-device-only", f"{build.CSRC}/delta.hip", "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    assert text.count("s_or_b64 exec, exec") > 100
    assert lost_writes(text) == []
