"""What the kernels' sources must not do, checked by reading them."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ojasx-vector-24x96_b200", "csrc")


def _code(path):
    """A source without its comments."""
    with open(path) as f:
        return re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)


def test_masks_of_shuffles_name_the_lanes_that_take_part():
    """__activemask() gives the lanes that happen to be together at that place, not those that a shuffle is meant for."""
    sources = glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))
    assert sources
    assert [os.path.basename(p) for p in sources if "__activemask" in _code(p)] == []


def test_every_wrapper_has_a_caller():
    """Device functions of the header of instruction wrappers are called by a kernel (or by one another)."""
    code = {os.path.basename(p): _code(p) for p in glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))}
    names = set(re.findall(r"\b(tc_\w+)\(", code["tc.cuh"]))
    assert len(names) > 20
    assert [n for n in sorted(names) if sum(len(re.findall(rf"\b{n}\b", text)) for text in code.values()) < 2] == []


def test_the_decode_has_no_workspace_for_other_types():
    import ctypes
    from ojasx_b200._lib import Q4Cache, lib
    c = Q4Cache(pool=4096, status=4096, turns=None, num_pages=1, page_size=16, kv_heads=2, q_heads=4, head_dim=128)
    size = [lib().ojasx_b200_q4kv_decode_workspace(ctypes.addressof(c), 1, 1, t) for t in (0, 1, 2, -1)]
    assert size[0] == size[1] > 0 and size[2:] == [0, 0]
