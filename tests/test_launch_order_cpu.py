"""Every kernel that lets its successor start early waits for its predecessor first (read from the sources)."""
import glob
import os
import re

from aegaeon_b200.build import CSRC

# Launched without the programmatic attribute: it begins when everything before it has completed.
PLAIN = {"decode_plan_kernel"}


def _functions():
    """(file, name, body) of every __global__ function."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        src = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"__global__", src):
            begin = src.index("{", src.index(")", src.index("kernel", m.end())))
            name = re.search(r"(\w*kernel)\s*\(", src[m.end():begin + 1]).group(1)
            depth, i = 0, begin
            while True:
                depth += {"{": 1, "}": -1}.get(src[i], 0)
                i += 1
                if depth == 0:
                    break
            yield os.path.basename(path), name, src[begin:i]


def test_kernels_wait_before_they_let_the_next_one_start():
    seen = set()
    for path, name, body in _functions():
        seen.add(name)
        for m in re.finditer(r"pdl_launch_dependents\(\)", body):
            assert name in PLAIN or "pdl_wait_primary()" in body[:m.start()], f"{path}: {name}"
    assert {"rotary_kernel", "write_int4_kernel", "gather_int4_kernel", "free_kernel", "compact_apply_kernel",
            "reshape_and_cache_vec_kernel", "decode_attn_kernel", "decode_attn_int4_kernel"} <= seen


def test_only_cache_writes_start_their_successor_before_the_wait():
    users = {name for _, name, body in _functions() if "pdl_enter_write" in body}
    assert users == {"write_int4_kernel", "reshape_and_cache_vec_kernel", "reshape_and_cache_warp_kernel",
                     "reshape_and_cache_elem_kernel"}
