"""What the kernels' host code must not do: a rule on the sources, no GPU needed."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pico-vllm_b200", "csrc")


def test_limits_of_shared_memory_are_set_in_one_place():
    """The limit belongs to a kernel, not to a launch: set to each call's own size it would be taken from under another thread's launch.  Only the
    function that raises it and never lowers it may set it."""
    where = {}
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh", ".h")):
            with open(os.path.join(CSRC, name)) as f:
                n = len(re.findall("cudaFuncAttributeMaxDynamicSharedMemorySize|FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES", f.read()))
            if n:
                where[name] = n
    assert where == {"common.cuh": 1}
