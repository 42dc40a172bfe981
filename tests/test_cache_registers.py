"""The attention kernels keep everything in registers: the compiler that builds them has stored and reloaded three registers of a spilled four,
which gave wrong scores.  Looked at in the built library, from the metadata of its code objects."""
import os
import re
import shutil
import subprocess

import pytest

from test_mfma_waits import _code_objects

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
READELF = shutil.which("llvm-readelf", path="/opt/rocm/llvm/bin:" + os.environ.get("PATH", ""))


@pytest.mark.skipif(READELF is None, reason="llvm-readelf is not there")
def test_no_attention_kernel_spills(tmp_path):
    found = {}
    for k, part in enumerate(_code_objects(os.path.join(ROOT, "aihwkit_amd", "lib", "librpu_amd.so"))):
        path = tmp_path / f"{k}.co"
        path.write_bytes(part)
        notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for kernel in re.split(r"\n  - ", notes)[1:]:
            name = re.search(r"\.name: +(\S+)", kernel)
            if name and re.search("8k_attend|14k_attend_mixed", name.group(1)):
                found[name.group(1)] = (int(re.search(r"\.vgpr_spill_count: +(\d+)", kernel).group(1)),
                                        int(re.search(r"\.private_segment_fixed_size: +(\d+)", kernel).group(1)))
    # five pairs of types; four widths in tiles of lines, three (beside 16-bit rows four) with few lines, three (floats: none) with both
    assert len(found) == 49, len(found)
    assert set(found.values()) == {(0, 0)}, {name: v for name, v in found.items() if v != (0, 0)}
