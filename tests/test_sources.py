"""What the kernels' sources may not contain."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "daisy_b200", "csrc")


def _code():
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        with open(path) as f:
            text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
        yield os.path.basename(path), re.sub(r"//[^\n]*", "", text)


def test_loads_of_global_memory_are_coherent():
    """Grids are launched as dependents and may be resident while the grids before them still write what they will read; the
    non-coherent path is defined only for memory that nobody writes while the kernel lives."""
    seen = 0
    for name, text in _code():
        seen += 1
        assert not re.search(r"ld\.global(\.\w+(::\w+)?)*\.nc\b", text) and "__ldg(" not in text, name
    assert seen >= 10
