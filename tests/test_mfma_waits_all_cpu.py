"""test_mfma_waits_cpu.py's check of early reads of matrix products' results, for products whose results are in
accumulation registers too, over every source with matrix products.  CPU only."""
import os
import re
import subprocess

import pytest

from nemotron_infer_amd import build
from tests import test_mfma_waits_cpu


def _wait_states(op):
    """4x4x4 products take two passes of the matrix core: five wait states, which the compiler keeps."""
    return 5 if "_4x4x4" in op else test_mfma_waits_cpu._wait_states(op)


def _regs(text):
    """Vector and accumulation registers that an instruction names, apart from one another."""
    out = {(f, int(r)) for f, r in re.findall(r"\b([va])(\d+)\b", text)}
    for f, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        out |= {(f, r) for r in range(int(a), int(b) + 1)}
    return out


def early_reads(asm):
    lines = [s for s in (re.sub(r";.*", "", x).strip() for x in asm.splitlines()) if s]
    labels = {s[:-1]: i for i, s in enumerate(lines) if re.fullmatch(r"\S+:", s)}
    found, products = [], 0
    for i, s in enumerate(lines):
        m = re.match(r"(v_mfma\S+) ([va]\[\d+:\d+\])", s)
        if not m:
            continue
        products += 1
        result, limit = _regs(m[2]), _wait_states(m[1])
        todo, seen = [(i + 1, 0)], set()
        while todo:
            j, d = todo.pop()
            if j >= len(lines) or d >= limit or (j, d) in seen:
                continue
            seen.add((j, d))
            t = lines[j]
            if t.endswith(":") or t.startswith("."):
                todo.append((j + 1, d))
            elif t.startswith("s_nop"):
                todo.append((j + 1, d + int(t.split()[1]) + 1))
            elif t.startswith("s_cbranch"):
                todo += [(labels[t.split()[1]], d + 1), (j + 1, d + 1)]
            elif t.startswith("s_branch"):
                todo.append((labels[t.split()[1]], d + 1))
            elif re.match(r"(v_|ds_|global_|buffer_|flat_)", t) and not t.startswith("v_mfma") and _regs(t) & result:
                found.append((s, t, d))
            elif not t.startswith("s_endpgm"):
                todo.append((j + 1, d + 1))
    return products, found


def test_the_check_sees_an_early_read_of_an_accumulation_register():
    body = "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], 0\ns_cbranch_scc0 L\ns_nop 7\nL:\n{}v_accvgpr_read_b32 v9, a3"
    assert len(early_reads(body.format(""))[1]) == 1
    assert not early_reads(body.format("s_nop 6\n"))[1]
    assert not early_reads(body.format("").replace("a3", "a4"))[1]
    assert not early_reads(body.format("s_nop 3\n").replace("16x16x32_bf16", "4x4x4_16b_bf16"))[1]
    assert len(early_reads(body.format("s_nop 2\n").replace("16x16x32_bf16", "4x4x4_16b_bf16"))[1]) == 1
    assert not early_reads("v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], 0\nv_add_f32_e32 v9, v3, v3\ns_endpgm")[1]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("source", [s for s in build.HIP_SOURCES
                                    if "mfma" in open(os.path.join(build.CSRC, s)).read()])
def test_no_early_reads(source, tmp_path):
    out = tmp_path / "kernels.s"
    subprocess.run([build.HIPCC, "-x", "hip", *build.HIP_FLAGS, "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True, capture_output=True, timeout=300)
    asm = out.read_text()
    products, found = early_reads(asm)
    assert products == len(re.findall(r"^\s*v_mfma", asm, re.M)) > 0 and not found, found[:4]
