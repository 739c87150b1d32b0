"""What the generated code of the encoder-layer operators has to keep, checked on the CPU (built with the library's flags)."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "hybrid_rag_system_amd", "csrc")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
FLAGS = ["--offload-arch=gfx950", "-O3", "-std=c++17", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
SOURCES = ["hrs_linear.hip", "hrs_attention.hip", "hrs_norm.hip"]

pytestmark = pytest.mark.skipif(not (os.path.exists(HIPCC) or shutil.which("hipcc")), reason="hipcc not installed")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """source -> the lines of its generated assembly (all sources at once)."""
    d = tmp_path_factory.mktemp("isa")
    jobs = [(s, d / (s + ".s")) for s in SOURCES]
    running = [subprocess.Popen([HIPCC] + FLAGS + ["--cuda-device-only", "-S", os.path.join(CSRC, s), "-o", str(o)], stderr=subprocess.DEVNULL) for s, o in jobs]
    assert all(p.wait() == 0 for p in running)
    return {s: o.read_text().splitlines() for s, o in jobs}


def _kernels(lines):
    """name -> [(is a label, text)]"""
    out, name, body = {}, None, []
    for line in lines:
        m = re.match(r"^(_Z\w+):", line)
        if m:
            name, body = m.group(1), []
        elif line.startswith(".Lfunc_end") and name:
            out[name], name = body, None
        elif name:
            t = line.split(";")[0].strip()
            if re.match(r"^\.LBB\S+:", t):
                body.append((True, t[:-1]))
            elif t and not t.startswith((".", "//")):
                body.append((False, t))
    return out


def _registers(text):
    regs = set()
    for kind, lo, hi in re.findall(r"\b([av])\[(\d+):(\d+)\]", text):
        regs.update((kind, n) for n in range(int(lo), int(hi) + 1))
    regs.update((kind, int(n)) for kind, n in re.findall(r"\b([av])(\d+)\b", text))
    return regs


@pytest.mark.parametrize("source", ["hrs_linear.hip", "hrs_attention.hip"])
def test_results_of_matrix_instructions_rest(code, source):
    """A matrix instruction's result is not interlocked for other vector instructions: 7 wait states after one of 16 x 16
    x 32, 11 after one of 32 x 32 x 16.  The compiler counts them, but has missed a read behind a branch (keys 27 and 31
    of every tile then had an older score).  Walked along every path from every such instruction."""
    checked = 0
    for name, body in _kernels(code[source]).items():
        labels = {t: i for i, (is_label, t) in enumerate(body) if is_label}
        for i, (is_label, text) in enumerate(body):
            if is_label or not text.startswith("v_mfma"):
                continue
            checked += 1
            need, result = 11 if "_32x32x16_" in text else 7, _registers(text.split(",")[0])
            paths, seen = [(i + 1, 0)], {}
            while paths:
                j, waited = paths.pop()
                while j < len(body) and waited < need and seen.get(j, need) > waited:
                    seen[j] = waited
                    is_label, ins = body[j]
                    j += 1
                    if is_label:
                        continue
                    op = ins.split()[0]
                    if op == "s_endpgm" or (op.startswith("v_mfma") and _registers(ins.split(",")[0]) == result):
                        break  # (the next instruction of the same sum is interlocked, and checked itself)
                    if not op.startswith(("v_mfma", "s_")):
                        assert not _registers(ins) & result, (name, text, ins, waited, need)
                    if op == "s_branch" or op.startswith("s_cbranch"):
                        paths.append((labels[ins.split()[-1]], waited + 1))
                        if op == "s_branch":
                            break
                    waited += int(ins.split()[1], 0) + 1 if op == "s_nop" else 1
    assert checked > 1000


@pytest.mark.parametrize("source", SOURCES)
def test_no_spills_and_no_packed_fp32(code, source):
    """A spill's scratch accesses count in vmcnt, which these kernels wait on with counts; packed fp32 instructions are
    switched off for the library."""
    spills = [line for line in code[source] if re.match(r"\s+\.vgpr_spill_count:\s+[1-9]", line)]
    assert not spills
    assert not [line for line in code[source] if re.search(r"\bv_pk_(add|mul|fma)_f32", line)]
