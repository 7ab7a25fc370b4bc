"""The attention kernels' assembly, as the Makefile's flags make it: where lanes that skipped
a branch come back, nothing is copied in front of the instruction that switches them on
again.  With more live registers than a kernel has, the compiler has put copies of live registers
(to accumulation registers and scratch) there; the lanes that had skipped the branch
kept stale values, addresses among them.  CPU only."""
import os
import re
import shlex
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "fast-llm_amd", "csrc")
COPY = re.compile(r"v_accvgpr_(write|read|mov)|scratch_(store|load)|v_mov_b(32|64)\w* v\S+ v\S+$")
ON_AGAIN = re.compile(r"s_or_b64 exec, exec")
OTHER_EXEC = re.compile(r"s_(xor|andn2|and|mov)_b64 exec|s_\w+_saveexec|s_cbranch|s_branch|s_endpgm|s_setpc")


def copies_at_joins(asm):
    """{kernel: [(label, copies)]}: copies between the label of a skipped branch's end and
    the instruction that switches the lanes on again."""
    lines = [x.split(";")[0].strip() for x in asm.split("\n")]
    joins = set(re.findall(r"s_cbranch_execz\s+(\.LBB\d+_\d+)", asm))
    found, kernel, label, copies = {}, None, None, []
    for t in lines:
        m = re.match(r"(_Z\w+):", t)
        if m:
            kernel, label = m.group(1), None
        elif t.startswith(".LBB"):
            label, copies = (t[:-1] if t[:-1] in joins else None), []
        elif label and ON_AGAIN.match(t):
            if copies:
                found.setdefault(kernel, []).append((label, copies))
            label = None
        elif OTHER_EXEC.match(t):
            label = None
        elif label and COPY.match(t.replace(",", "")):
            copies.append(t)
    return found


def test_the_check_finds_copies():
    asm = """_Zkernel:
\ts_and_saveexec_b64 s[0:1], vcc
\ts_cbranch_execz .LBB0_2
\tv_mov_b32_e32 v1, v2
.LBB0_2:                                ; the end of the branch
\tv_add_u32_e32 v3, v1, v2
%s
\ts_or_b64 exec, exec, s[0:1]
\tv_mov_b32_e32 v4, v5
\ts_endpgm
"""
    assert copies_at_joins(asm % "\ts_nop 0") == {}
    for bad in ("\tv_accvgpr_write_b32 a176, v173", "\tscratch_store_dword off, v9, s33 offset:4", "\tv_mov_b32_e32 v7, v8"):
        assert copies_at_joins(asm % bad) == {"_Zkernel": [(".LBB0_2", [bad.strip()])]}


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_no_copies_at_joins(tmp_path):
    jobs = []
    for name in ("flh_attn_dec", "flh_attn_pre"):
        plan = subprocess.run(["make", "-n", "-B", "-C", CSRC, "BUILD=" + str(tmp_path), str(tmp_path / (name + ".o"))],
                              check=True, capture_output=True, text=True).stdout
        line = next(x for x in plan.split("\n") if "hipcc" in x and name + ".hip" in x)
        args = shlex.split(line[line.index("/opt/rocm"):line.index(" 2>&1")])
        out = tmp_path / (name + ".s")
        args[args.index("-o") + 1] = str(out)
        args[args.index("-c")] = "-S"
        jobs.append((out, subprocess.Popen(args + ["--cuda-device-only"], cwd=CSRC, stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)))
    for out, p in jobs:
        assert p.wait(timeout=600) == 0
        asm = out.read_text()
        assert asm.count("s_or_b64 exec, exec") > 100 and "k_attn_join" in asm
        assert copies_at_joins(asm) == {}
