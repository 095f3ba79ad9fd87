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


def test_a_steps_lengths_are_read_through_l2_before_the_wait():
    """What a step uploads is read in front of the wait for the kernels before, where only `ld_step` may read it: no entry,
    group or range of attention over shared prefixes is found by a plain load of the step's arrays."""
    text = code("shared_prefix.cuh")
    reads = body(text, "struct Groups")
    assert re.findall(r"ld_step\((\w+) \+ g\)", reads) == ["off", "prefix"]
    for name in ("group_of", "raw_of", "token_of", "Entry entry_of", "Groups hold_groups", "Range find_range"):
        inside = body(text, name + "(")
        arrays = r"(?:cu_q|ctx_len|prefix_len|group_off|block_table|(?:gs?)\.(?:off|prefix))"
        assert not re.search(arrays + r"\s*\[", inside), name
        for use in re.finditer(arrays + r"\s*\+", inside):
            assert inside[:use.start()].endswith("ld_step(b."), name
