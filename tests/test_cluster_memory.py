"""Another block's shared memory exists once that block runs, which only a barrier of the cluster establishes: every kernel has to pass
one before it forms a cluster address.  Read from the sources, as breaking the rule may fault the GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gpu-experiments_b200", "csrc")
BARRIER = re.compile(r"cluster_sync_all\s*\(|cluster_wait\s*\(|barrier\.cluster\.wait")


def kernels():
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cu"):
            continue
        text = open(os.path.join(CSRC, name)).read()
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
        for body in re.split(r"__global__", text)[1:]:
            if "map_to_cta(" in body:
                yield name, re.search(r"(\w+)\s*\(", re.sub(r"__\w+__\s*\([^;{]*?\)\s*", "", body)).group(1), body


FOUND = list(kernels())


def test_some_kernels_are_looked_at():
    assert {"router.cu", "gemm.cu", "block128_gemm.cu"} <= {f for f, _, _ in FOUND}


@pytest.mark.parametrize("file,kernel,body", FOUND, ids=[f"{f}:{k}" for f, k, _ in FOUND])
def test_barrier_before_remote_shared_memory(file, kernel, body):
    assert BARRIER.search(body[:body.index("map_to_cta(")]), f"{file}: {kernel} uses another block's shared memory before a cluster barrier"
