"""What inline assembly writes beside its operands is declared, so that the compiler keeps nothing there."""
import glob
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_assembly_that_writes_m0_says_so():
    found = 0
    for path in glob.glob(os.path.join(ROOT, "aihwkit_amd", "csrc", "*.h")) + glob.glob(os.path.join(ROOT, "aihwkit_amd", "csrc", "*.hip")):
        for statement in re.findall(r"\basm\b[^;]*;", open(path).read()):
            if re.search(r"s_mov_b32 m0,", statement):
                found += 1
                assert statement.count('"m0"') == 1, (path, statement)
    assert found >= 1
