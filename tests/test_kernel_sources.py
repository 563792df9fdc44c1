"""Rules that the kernels' sources keep and that no run can be relied on to show."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "etalii", "dllm_b200", "csrc")


def _code(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name), encoding="utf-8") as handle:
        return re.sub(r"//[^\n]*", "", handle.read())


def test_blocks_that_read_each_others_memory_meet_in_order():
    """attention_shared's blocks read the others' shared memory, and rows of scratch that another block of the cluster has written,
    up to a barrier of the cluster: each of its barriers orders memory."""
    code = _code("attention_shared.cu")
    assert "barrier.cluster.arrive" in code
    assert not re.search(r"barrier\.cluster\.arrive(?!\.release)", code) and not re.search(r"barrier\.cluster\.wait(?!\.acquire)", code)
