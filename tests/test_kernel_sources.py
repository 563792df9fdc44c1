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


def _kernel(code, name):
    """The body of the kernel `name`."""
    at = code.index("{", re.search(rf"\b{name}\s*\(", code).end())
    depth = 0
    for i in range(at, len(code)):
        depth += {"{": 1, "}": -1}.get(code[i], 0)
        if depth == 0:
            return code[at:i + 1]
    raise AssertionError(f"{name} does not end")


def test_what_attention_reads_ahead_of_its_wait_is_written_by_kernels_that_are_over():
    """Attention reads positions, page tables and cached rows of earlier steps ahead of its wait. The kernels that write them
    wait for the one in front and do not let the one behind start early."""
    for source, kernel in (("beam_reorder.cu", "reorder_kernel"), ("elementwise.cu", "decode_advance_kernel")):
        body = _kernel(_code(source), kernel)
        assert "pdl_wait()" in body and "launch_dependents" not in body, (source, kernel)


def test_shared_arrays_that_are_read_in_16_bytes_are_aligned_to_them():
    """attention_shared: an array of floats in shared memory has no alignment but a float's unless it is given one."""
    code = _code("attention_shared.cu")
    read = set(re.findall(r"\bfour\((sm_\w+)", code))
    read |= set(re.findall(r"reinterpret_cast<(?:const )?(?:float4|ulonglong2|uint4)\s*\*>\(\s*&?\s*(sm_\w+)", code))
    assert {"sm_fade", "sm_shift", "sm_p"} <= read
    declarations = re.findall(r"__shared__ ([^;]*);", code)
    for name in read:
        holding = [d for d in declarations if re.search(rf"\b{name}\s*\[", d)]
        assert holding and all("__align__(16)" in d for d in holding), name
