"""The shared-prefix attention's S^T chains keep their accumulators in VGPRs by inline assembly, as the
sparse attention's do: no instruction may touch an accumulator while its chain is in flight, on any path
of the compiled code (the walk of test_isa_chains). CPU only; needs hipcc."""
import os
import re
import subprocess

import pytest

from dsa_triton_ascend_amd import build

from .test_isa_chains import CSRC, HIPCC, chain_violations, chains_by_kernel


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="hipcc not available")
def test_chains_never_touched_in_flight(tmp_path):
    asm = tmp_path / "listing.s"
    cmd = [HIPCC, *build.COMMON, "-x", "hip", "-S", "--cuda-device-only", os.path.join(CSRC, "prefix_attn.hip"), "-o", str(asm)]
    p = subprocess.run(cmd, capture_output=True, text=True)
    assert p.returncode == 0, p.stderr[-2000:]
    lines = asm.read_text().splitlines()
    chains, bad = chain_violations(lines)
    found = {n: c for n, c in chains_by_kernel(lines).items() if "prefix_attn_kernel" in n}
    # per type and D: 128 head rows with the first tile's chain and the loop's, 64 and 32 with one each
    assert len(found) == 6 and min(found.values()) >= 4 and sum(found.values()) == chains
    assert not bad, f"accumulator touched while its chain is in flight: {bad[:5]}"
    # every direct-to-LDS load takes its LDS address from a scalar register
    assert not [l for l in lines if re.search(r"s_mov_b32 m0, v", l)]
