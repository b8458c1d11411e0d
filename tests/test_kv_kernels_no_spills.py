"""The rotary, append and cache attention kernels keep what they hold in registers: compiled to gfx950 assembly, each
stays within the registers of the waves it is launched for (two a SIMD for the attention kernels), and none spills a
VGPR to scratch memory, but for the attention of 128 channels: it runs at the edge of the register file and keeps some
values there around its loops, never in the steps over whole tiles, where its time goes.  CPU only (hipcc
cross-compiles)."""
import os
import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "pasa_amd" / "csrc"
HIPCC = os.environ.get("HIPCC", shutil.which("hipcc") or "/opt/rocm/bin/hipcc")

# kernel -> (instantiations, most VGPRs)
AT_THE_EDGE = r"kv_attn_(rows|tiles)\S*Li128E"
KERNELS = {
    "kv_attn.hip": {"kv_attn_rows": (8, 256), "kv_attn_tiles": (12, 256), "kv_attn_join": (2, 128)},
    "kv_append.hip": {"kv_append": (3, 128)},
    "rope_axes.hip": {"rope_axes_vec": (6, 128), "rope_axes_scalar": (3, 64)},
}


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
@pytest.mark.parametrize("src", sorted(KERNELS))
def test_no_spills(src, tmp_path):
    out = tmp_path / (src + ".s")
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", str(CSRC / src), "-o", str(out)],
                   check=True, capture_output=True)
    asm = out.read_text()
    seen = dict.fromkeys(KERNELS[src], 0)
    for block in re.split(r"\n\s+- \.", asm):
        name = re.search(r"\.name:\s+(\S+)", block)
        if not name:
            continue
        num = lambda key: int(re.search(r"\.%s:\s+(\d+)" % key, block).group(1))
        for kernel, (_, most) in KERNELS[src].items():
            if re.search(r"\d%s[IE]" % kernel, name.group(1)):
                seen[kernel] += 1
                if not re.search(AT_THE_EDGE, name.group(1)):
                    assert num("vgpr_spill_count") == 0, name.group(1)
                assert num("vgpr_count") <= most, (name.group(1), num("vgpr_count"))
    assert seen == {k: n for k, (n, _) in KERNELS[src].items()}, seen
    # A step over a whole tile of 128 channels is one block of 64 MFMAs.
    for body in re.finditer(r"\n(_ZN4pasa\S*kv_attn_tiles\S*Li128E\S*):.*?s_endpgm", asm, re.S):
        steps = [b for b in re.split(r"\n(?=\.LBB\S+:)", body.group(0)) if b.count("v_mfma") >= 64]
        assert steps and not any("scratch_" in b for b in steps), body.group(1)


@pytest.mark.skipif(not Path(HIPCC).exists(), reason="hipcc not available")
def test_barriers_wait_for_lds_writes(tmp_path):
    """LDS answers a wave in order: a barrier may leave N LDS operations in flight only where the wave's last N are reads,
    or its writes may come behind what other waves read past the barrier."""
    out = tmp_path / "kv_attn.s"
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "--cuda-device-only", "-S", str(CSRC / "kv_attn.hip"), "-o", str(out)],
                   check=True, capture_output=True)
    lines = [line.split(";")[0].strip() for line in out.read_text().splitlines()]
    open_waits = 0
    for i, line in enumerate(lines):
        if line != "s_barrier":
            continue
        wait = next(j for j in range(i - 1, -1, -1) if "lgkmcnt" in lines[j] or lines[j].startswith("ds_"))
        left = re.search(r"lgkmcnt\((\d+)\)", lines[wait])
        assert left, (i, lines[wait])
        left = int(left.group(1))
        if left:
            ops = [x for x in lines[max(wait - 400, 0):wait] if x.startswith("ds_")][-left:]
            assert all(x.startswith("ds_read") for x in ops), (i, ops)
            open_waits += 1
    assert open_waits
