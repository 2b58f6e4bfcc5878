"""A rule of the kernels that come up while the one before still runs, kept by their sources."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(__file__), "..", "sketchpad_b200", "csrc")


def test_overlapped_kernels_read_with_ordinary_loads():
    """Non-coherent loads are defined only for data that nobody writes while the kernel lives."""
    seen = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu"))):
        with open(path) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        if "griddepcontrol.launch_dependents" not in text:
            continue
        seen += 1
        assert text.count("griddepcontrol.wait") == text.count("griddepcontrol.launch_dependents")
        for word in ("__ldg(", "ld.global.nc", "__restrict__"):
            assert word not in text, (os.path.basename(path), word)
    assert seen == 4
