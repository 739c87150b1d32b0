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


def _walk(lines, need_of):
    """Every read of a matrix instruction's result along every path behind it -> (instructions, reads that come early)."""
    checked, early = 0, []
    for name, body in _kernels(lines).items():
        labels = {t: i for i, (is_label, t) in enumerate(body) if is_label}
        for i, (is_label, text) in enumerate(body):
            if is_label or not text.startswith("v_mfma"):
                continue
            checked += 1
            need, result = need_of(text), _registers(text.split(",")[0])
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
                        break
                    if not op.startswith(("v_mfma", "s_")) and _registers(ins) & result:
                        early.append((name, text, ins, waited, need))
                        break
                    if op == "s_branch" or op.startswith("s_cbranch"):
                        paths.append((labels[ins.split()[-1]], waited + 1))
                        if op == "s_branch":
                            break
                    waited += int(ins.split()[1], 0) + 1 if op == "s_nop" else 1
    return checked, early


_PROBE = """
#include <hip/hip_runtime.h>
typedef __bf16 x8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16 __attribute__((ext_vector_type(16)));
__global__ void probe_32x32x16(const x8* a, float* out) {
    f16 c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[threadIdx.x], a[threadIdx.x + 64], (f16)(0.f), 0, 0, 0);
    out[threadIdx.x] = c[0] + c[15];
}
__global__ void probe_16x16x32(const x8* a, float* out) {
    f4 c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[threadIdx.x], a[threadIdx.x + 64], (f4)(0.f), 0, 0, 0);
    out[threadIdx.x] = c[0] + c[3];
}
"""


@pytest.fixture(scope="module")
def wait_states(tmp_path_factory):
    """Shape -> wait states that this compiler itself puts between such an instruction and the first vector read of its
    result, in a straight line."""
    d = tmp_path_factory.mktemp("probe")
    (d / "probe.hip").write_text(_PROBE)
    subprocess.run([HIPCC] + FLAGS + ["--cuda-device-only", "-S", str(d / "probe.hip"), "-o", str(d / "probe.s")], check=True, stderr=subprocess.DEVNULL)
    found = {}
    for body in _kernels((d / "probe.s").read_text().splitlines()).values():
        at = next(i for i, (_, t) in enumerate(body) if t.startswith("v_mfma"))
        result, waited = _registers(body[at][1].split(",")[0]), 0
        for _, ins in body[at + 1 :]:
            op = ins.split()[0]
            if not op.startswith("s_") and _registers(ins) & result:
                break
            waited += int(ins.split()[1], 0) + 1 if op == "s_nop" else 1
        found[re.search(r"\d+x\d+x\d+", body[at][1]).group()] = waited
    return found


def test_wait_states_of_the_compiler(wait_states):
    """8 passes of four cycles and 3 more for the 32 x 32 x 16 product, 4 and 3 for the 16 x 16 x 32 one, and the read's own."""
    assert wait_states == {"32x32x16": 12, "16x16x32": 8}


@pytest.mark.parametrize("source", ["hrs_linear.hip", "hrs_attention.hip"])
def test_results_rest_as_long_as_the_compiler_waits(code, wait_states, source):
    checked, early = _walk(code[source], lambda text: wait_states[re.search(r"\d+x\d+x\d+", text).group()])
    assert checked > 1000 and not early, early[:3]


def test_walk_catches_an_early_read():
    """The walk itself: a read behind a branch, one wait state too early, and the same one further on."""
    text = "_Z1kPf:\n v_mfma_f32_32x32x16_bf16 v[0:15], v[16:19], v[20:23], 0\n s_cbranch_scc1 .LBB0_2\n s_nop 11\n v_add_f32_e32 v20, v0, v1\n s_endpgm\n.LBB0_2:\n s_nop %d\n v_add_f32_e32 v20, v0, v15\n s_endpgm\n.Lfunc_end0:\n"
    assert _walk((text % 10).splitlines(), lambda t: 12) == (1, [])
    checked, early = _walk((text % 9).splitlines(), lambda t: 12)
    assert checked == 1 and early[0][3:] == (11, 12)


def test_flags_are_the_librarys():
    """FLAGS and SOURCES against what make would run."""
    plan = subprocess.run(["make", "-n", "-B", "-C", CSRC], check=True, capture_output=True, text=True).stdout
    for source in SOURCES:
        line = next(l for l in plan.splitlines() if f"-c {source} " in l)
        assert [f for f in line.split()[1:] if f not in ("-fPIC", "-Wall", "-Wno-unused-function", "-c", source, "-o", source.replace(".hip", ".o"))] == FLAGS, line


def test_other_kernels_have_no_matrix_instructions():
    """What SOURCES leaves out of the encoder of other geometries has nothing to wait for."""
    with open(os.path.join(CSRC, "hrs_encoder_any.hip")) as f:
        assert "mfma" not in f.read()
