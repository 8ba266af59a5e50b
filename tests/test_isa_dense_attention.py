"""The dense attention's S and dP products are inline-asm MFMAs with accumulators in VGPRs and one operand in
AGPRs (dense_attn.hpp: mfma32_va*), which the compiler does not see in flight: it adds none of the wait states that
it would for its own. In the compiled code (gfx950, device code only, as assembly) of both files that hold them:

- from each such MFMA on, on every path, no other vector instruction names its accumulator until the next MFMA
  adds to it or 16 wait states of s_nop have passed (8 passes: 12 are needed);
- no operand is written by a VALU instruction less than two wait states before.

CPU only; needs hipcc."""
import os
import re
import subprocess

import pytest

from dsa_triton_ascend_amd import build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
CSRC = os.path.join(ROOT, "dsa_triton_ascend_amd", "csrc")
DRAIN = 16
BEFORE = 2

_MFMA = re.compile(r"v_mfma_f32_32x32x16_(?:bf16|f16) ([va]\[\d+:\d+\]), ([va]\[\d+:\d+\]), ([va]\[\d+:\d+\]), (\S+)")


def _regs(text):
    out = set()
    for kind, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", text):
        out |= {(kind, i) for i in range(int(a), int(b) + 1)}
    for kind, a in re.findall(r"(?<![\w\[:])([va])(\d+)\b", text):
        out.add((kind, int(a)))
    return out


def parse(lines):
    """Instructions (text, in an asm statement, kernel, line) and the index that each label stands at"""
    ins, labels, in_asm, name = [], {}, False, None
    for i, line in enumerate(lines):
        m = re.match(r"^(\.?\w+):", line)
        if m:
            labels[m.group(1)] = len(ins)
            if m.group(1).startswith("_Z"):
                name = m.group(1)
            continue
        if "ASMSTART" in line or "ASMEND" in line:
            in_asm = "ASMSTART" in line
            continue
        text = line.split(";")[0].strip()
        if text and not text.startswith((".", "%")):
            ins.append((text, in_asm, name, i + 1))
    return ins, labels


def touched_in_flight(ins, labels, start, acc):
    """The first instruction on some path from `start` that names a register of acc before its MFMA is through"""
    regs = _regs(acc)
    stack, seen = [(start, 0)], set()
    while stack:
        j, nops = stack.pop()
        while j < len(ins):
            if (j, nops) in seen:
                break
            seen.add((j, nops))
            text = ins[j][0]
            op = text.split()[0]
            m = _MFMA.match(text)
            if m and m.group(4) == acc:   # adds to it (its own result is looked at from there)
                if not _regs(m.group(2) + m.group(3)) & regs:
                    break
                return ins[j]
            if op == "s_nop":
                nops += int(text.split()[1]) + 1
                if nops >= DRAIN:
                    break
            elif not op.startswith("s_") and _regs(text.partition(" ")[2]) & regs:
                return ins[j]
            elif op == "s_branch":
                j = labels[text.split()[1]]
                continue
            elif op.startswith("s_cbranch"):
                stack.append((labels[text.split()[1]], nops))
            elif op in ("s_endpgm", "s_setpc_b64"):
                break
            j += 1
    return None


def written_just_before(ins, k, uses):
    """A VALU write of a register in `uses` less than BEFORE wait states ahead of instruction k, in line"""
    wait, j = 0, k - 1
    while j >= 0 and wait < BEFORE:
        text = ins[j][0]
        op = text.split()[0]
        if op == "s_nop":
            wait += int(text.split()[1]) + 1
        else:
            if op.startswith("v_") and not op.startswith(("v_mfma", "v_cmp")):
                operands = text.partition(" ")[2].split(",")
                out = operands[0] + ("," + operands[1] if "swap" in op else "")
                if _regs(out) & uses:
                    return ins[j]
            m = _MFMA.match(text)
            if m:
                uses = uses - _regs(m.group(1))
            wait += 1
        j -= 1
    return None


def check(lines):
    """Asm MFMAs of each kernel, and the faults (line, instruction, the MFMA)"""
    ins, labels = parse(lines)
    counts, bad = {}, []
    for k, (text, in_asm, name, line) in enumerate(ins):
        m = _MFMA.match(text)
        if not (m and in_asm):
            continue
        counts[name] = counts.get(name, 0) + 1
        uses = _regs(",".join(m.group(i) for i in (2, 3, 4)))
        for fault in (touched_in_flight(ins, labels, k + 1, m.group(1)), written_just_before(ins, k, uses)):
            if fault:
                bad.append((fault[3], fault[0], text))
    return counts, bad


def test_the_check_itself():
    first = ["_Zk:", "\t;;#ASMSTART", "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[20:23], a[0:3], 0", "\t;;#ASMEND"]
    last = ["\t;;#ASMSTART", "\tv_mfma_f32_32x32x16_bf16 v[0:15], v[24:27], a[4:7], v[0:15]", "\ts_nop 15", "\t;;#ASMEND"]
    use, end = ["\tv_mov_b32_e32 v40, v5"], ["\ts_endpgm"]
    assert check(first + last + use + end) == ({"_Zk": 2}, [])
    assert len(check(first + use + last + end)[1]) == 1
    assert len(check(first + last[:2] + ["\ts_nop 7", "\t;;#ASMEND"] + use + end)[1]) == 1
    branch = ["\ts_cbranch_vccz .L1"]
    assert len(check(first + branch + last + end + [".L1:"] + use + end)[1]) == 1
    write = ["\tv_accvgpr_write_b32 a5, v40"]
    assert len(check(first + write + last + end)[1]) == 1
    assert check(first + write + ["\ts_nop 1"] + last + end)[1] == []
    clear = ["\tv_mov_b32_e32 v3, 0"]
    assert len(check(first[:1] + clear + last + end)[1]) == 1     # a chain that starts from values
    assert check(first[:1] + clear + first[1:] + last + end)[1] == []   # overwritten, not read


# kernels with such chains, per file: instances and the least number of these MFMAs in each
EXPECTED = {"dense_attn.hip": {"dense_attn_kernel": (12, 8)},
            "dense_grad.hip": {"dense_keys_kernel": (12, 8), "dense_queries_kernel": (6, 8)}}


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
@pytest.mark.parametrize("source", sorted(EXPECTED))
def test_accumulators_in_flight_are_left_alone(source, tmp_path):
    asm = tmp_path / "listing.s"
    extra = ["-fno-honor-nans"] if source in build.NO_NANS else []
    p = subprocess.run([HIPCC, *build.COMMON, *extra, "-x", "hip", "-S", "--cuda-device-only", os.path.join(CSRC, source), "-o",
                        str(asm)], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr[-2000:]
    counts, bad = check(asm.read_text().splitlines())
    for kernel, (instances, least) in EXPECTED[source].items():
        got = [n for name, n in counts.items() if re.search(rf"\d{kernel}I", name)]
        assert len(got) == instances and min(got) >= least, f"{kernel}: MFMAs per instance {got}"
    assert not bad, f"accumulators or operands in flight: {bad[:5]}"
