"""What the kernels' sources promise about memory that other blocks write, and no run would show reliably."""

import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "somi_inference_b200", "csrc")


def code(name):
    """A source without its comments."""
    with open(os.path.join(CSRC, name), encoding="utf-8") as f:
        return re.sub(r"//[^\n]*", "", f.read())


def body(text, start):
    """The text from `start` to the end of the block that begins behind it."""
    at = text.index("{", text.index(start))
    depth, i = 0, at
    while True:
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        i += 1
        if depth == 0:
            return text[at:i]


def test_another_blocks_shared_memory_is_touched_behind_a_cluster_barrier():
    """A block of a cluster may not have begun when its neighbour has: the first access to another block's shared memory stands
    behind a barrier of the cluster, in every kernel that makes one."""
    found = 0
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith((".cu", ".cuh")):
            continue
        text = code(name)
        for kernel in re.finditer(r"__global__[^;{]*?\b(\w+_kernel)\s*\(", text):
            inside = body(text[kernel.start():], kernel.group(0))
            if "map_shared_rank" not in inside:
                continue
            found += 1
            before = inside[:inside.index("map_shared_rank")]
            assert "cluster.sync()" in before or ("cluster.barrier_arrive()" in before and "cluster.barrier_wait(" in before), (
                name, kernel.group(1))
    assert found >= 4
