"""What the compiler cannot check of the kernels' inline assembly: an instruction that writes M0 says so among its clobbers."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "ridgefill-data_amd" / "csrc"


def test_assembly_that_writes_m0_declares_it():
    seen = 0
    for f in sorted(CSRC.glob("*.h*")):
        for m in re.finditer(r"asm\s*volatile\s*\((.*?)\);", f.read_text(), re.S):
            if re.search(r"\bs_\w+ m0,", m.group(1)):
                seen += 1
                assert '"m0"' in m.group(1), (f.name, m.group(1))
    assert seen
