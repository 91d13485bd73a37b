"""A vector, LDS or memory instruction must not read a matrix product's result before the product has
passed through the matrix core: the compiler puts instructions or waits between the two, but leaves
them out where a branch lies between (seen in the paged decode kernel: a running maximum taken from half
of a score's sum, which changed the last bits of outputs from run to run).  This compiles the sources
for gfx950 with the library's own flags (device code only, to assembly) and follows every path from
each product for the instructions that the compiler itself keeps where it does see the dependence.
CPU only."""
import os
import re
import subprocess

import pytest

from nemotron_infer_amd import build


def _wait_states(op):
    return 12 if "32x32" in op else 8


def _regs(text):
    out = {int(r) for r in re.findall(r"\bv(\d+)", text)}
    for a, b in re.findall(r"\bv\[(\d+):(\d+)\]", text):
        out |= set(range(int(a), int(b) + 1))
    return out


def early_reads(asm):
    """(products, [(product, the instruction that reads it early, instructions between)])."""
    lines = [s for s in (re.sub(r";.*", "", x).strip() for x in asm.splitlines()) if s]
    labels = {s[:-1]: i for i, s in enumerate(lines) if re.fullmatch(r"\S+:", s)}
    found, products = [], 0
    for i, s in enumerate(lines):
        m = re.match(r"(v_mfma\S+) (v\[\d+:\d+\])", s)
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


def test_the_check_sees_an_early_read():
    body = "v_mfma_f32_16x16x32_bf16 v[0:3], v[4:7], v[8:11], 0\ns_cbranch_scc0 L\ns_nop 7\nL:\n{}v_max_f32_e32 v9, v3, v3"
    assert len(early_reads(body.format(""))[1]) == 1
    assert not early_reads(body.format("s_nop 6\n"))[1]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="hipcc not installed")
@pytest.mark.parametrize("source,least", [("sdpa_decode_paged.hip", 36), ("sdpa_prefill.hip", 300)])
def test_no_early_reads(source, least, tmp_path):
    out = tmp_path / "kernels.s"
    subprocess.run([build.HIPCC, "-x", "hip", *build.HIP_FLAGS, "--cuda-device-only", "-S",
                    os.path.join(build.CSRC, source), "-o", str(out)], check=True, capture_output=True, timeout=300)
    products, found = early_reads(out.read_text())
    assert products >= least and not found, found[:4]
