"""The delta rule's loads into LDS are written in assembly, whose waits are the source's own: what the compiler puts around them is
looked at here, in the assembly of a build for the GPU (no GPU needed)."""
from __future__ import annotations

import re
import subprocess

import pytest

from flyguy_amd.build import PKG, compile_flags, hipcc

WAIT = 5                                 # wait states from a vector instruction that writes a scalar register to a load that reads it


def scalars(text):
    """The scalar registers that operands name."""
    out = set()
    for a, b, one in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", text):
        out |= {int(one)} if one else set(range(int(a), int(b) + 1))
    return out


def functions(text):
    """Each function's instructions and labels, in order."""
    body, name = None, None
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if m := re.match(r"(_ZN\w+):$", line):
            name, body = m[1], []
        elif body is not None and line.startswith(".Lfunc_end"):
            yield name, body
            body = None
        elif body is not None and (re.match(r"\.LBB\w+:", line) or re.match(r"[a-z]\w+(\s|$)", line)):
            body.append(line)


def too_early(body):
    """(instruction, load) pairs where a vector instruction writes a scalar register of a load into LDS within the wait states."""
    label = {x[:-1]: i for i, x in enumerate(body) if x.endswith(":")}
    jumps = {}
    for i, x in enumerate(body):
        if (m := re.match(r"s_c?branch\w*\s+(\.LBB\w+)", x)):
            jumps.setdefault(m[1], []).append(i)
    bad, loads = [], 0

    def back(i, used, states, load, seen):
        """What may run before instruction i, `states` wait states before the load."""
        while i >= 0 and states < WAIT:
            x = body[i]
            if x.endswith(":"):
                for j in jumps.get(x[:-1], []):
                    if (j, states) not in seen:
                        seen.add((j, states))
                        back(j, used, states, load, seen)
            else:
                op, _, rest = x.partition(" ")
                if op in ("s_branch", "s_endpgm", "s_setpc_b64") and body[i + 1].endswith(":") and (i, states) not in seen:
                    return                                # (nothing falls through it)
                written = rest.split(",")[:2 if "_co_" in op or "div_scale" in op else 1]
                if op.startswith("v_") and scalars(",".join(written)) & used:
                    bad.append((x, load))
                states += int(rest) + 1 if op == "s_nop" else 1
            i -= 1

    for i, x in enumerate(body):
        if x.startswith("global_load_lds") or (x.startswith("buffer_load") and x.endswith("lds")):
            loads += 1
            back(i - 1, scalars(x), 0, x, set())
    assert all(x in label for x in jumps)
    return bad, loads


def test_the_search_finds_what_it_looks_for():
    for before, want in ((["v_readfirstlane_b32 s4, v1"], 1), (["v_readfirstlane_b32 s4, v1", "s_nop 4"], 0), (["v_readlane_b32 s5, v1, 3", "s_nop 2"], 1),
                         (["v_add_co_u32_e64 v1, s[4:5], v2, v3"], 1), (["v_cndmask_b32_e64 v1, v2, v3, s[4:5]"], 0),
                         (["v_readfirstlane_b32 s6, v1"], 0), (["s_add_u32 s4, s4, s6"], 0), (["v_add_u32 v4, s4, v5"], 0),
                         (["v_readfirstlane_b32 s4, v1", "s_branch .LBB0_2", ".LBB0_1:", "s_endpgm", ".LBB0_2:"], 1),
                         (["v_readfirstlane_b32 s4, v1", "s_endpgm", ".LBB0_2:"], 0)):
        bad, loads = too_early(before + ["s_mov_b32 m0, s9", "global_load_lds_dwordx4 v7, s[4:5]"])
        assert (len(bad), loads) == (want, 1), before


def test_no_load_reads_its_base_too_early(tmp_path):
    try:
        cc = hipcc()
    except RuntimeError:
        pytest.skip("no compiler here")
    out = tmp_path / "delta.s"
    subprocess.run([cc, *compile_flags(), "-S", "--cuda-device-only", str(PKG / "csrc" / "memory_delta.hip"), "-o", str(out)], check=True,
                   capture_output=True)
    loads, m0 = 0, []
    for name, body in functions(out.read_text()):
        bad, n = too_early(body)
        assert not bad, (name, bad[:3])
        loads += n
        # m0 is written for these loads alone, and exec is put back right after each
        for i, x in enumerate(body):
            if x.startswith("global_load_lds"):
                m0 += [i - 2]
                assert body[i - 2].startswith("s_mov_b32 m0,") and body[i - 1].startswith("s_and_saveexec_b64"), body[i - 2:i + 2]
                held = body[i - 1].split()[1].rstrip(",")
                assert body[i + 1] == f"s_mov_b64 exec, {held}", body[i - 2:i + 2]
        assert sum("m0" in x for x in body) == n, name
    assert loads > 100
