"""What the kernels' sources may not contain."""
import re
from pathlib import Path

SRC = Path(__file__).resolve().parent.parent / "src"


def _code(path):
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


def test_kernels_that_start_early_load_coherently():
    """A grid launched with programmatic serialization is there while the kernel before it still writes: loads by the non-coherent path, which may also be moved above the wait, are not for what that one writes."""
    files = [p for p in SRC.rglob("*.cu*") if re.search(r"pdl_begin\(\)|griddepcontrol\.wait", _code(p))]
    assert len(files) > 5
    for p in files:
        assert not re.search(r"__ldg\s*\(|ld\.global\.nc|ld\.global\.L1::no_allocate\.nc", _code(p)), p
